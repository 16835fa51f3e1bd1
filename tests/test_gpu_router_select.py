"""ops.router_select (scores, balance bias, groups, top-k, renormalised weights) against the same selection in
float64: ids equal, weights and gradients within float32 roundings.

Tolerances, derived: a weight is formed from scores with relative errors of at most 2^-21 (the row's maximum
subtracted, one exponential, one reciprocal; a softmax sum over C terms adds C 2^-24 in the worst order, 2^-18 for
64 lanes' sums of 65) and a sum and a quotient of such scores; a gradient from two products and one difference of such
terms: 2^-16 of the largest term of its row bounds both."""

import pytest
import torch

from helpers import gen

TOL = 2.0 ** -16


# A group's score is a sum of two scores in float64: exp (1 ulp), 1 + e, the quotient, the bias and the sum round
# it by at most 8 2^-53 of magnitudes below 2.  Two groups whose scores differ by less than this bound are not told
# apart by float64, and either may stay.  (Sums of scores around one logit come this close: with z = z0 + m 2^-25 two
# pairs with equal m + m' differ by their second derivative times 2^-50.)
GROUP_TIE = 2.0 ** -49


def reference(z, k, S=0, score="softmax", bias=None, G=1, g=None, best=2, renorm=True, scale=1.0, dw=None, got=None):
    """(idx, w, dz or None) on the CPU in float64; masked logits (-inf) come after every other.  ``got``: the
    kernel's ids, which say which of two groups stays where float64 does not tell them apart."""
    z = z.detach().cpu().double().requires_grad_(dw is not None)
    R, C = z.shape
    n, g = C - S, G if g is None else g
    best = min(best, n // G)
    body = z[:, S:]
    s = torch.softmax(body, 1) if score == "softmax" else torch.sigmoid(body)
    key = s.detach().clone() if bias is not None or (G > g and best == 2) else body.detach().clone()
    if bias is not None:
        key = key + bias.cpu().double()[S:]
    key = torch.where(body.detach() == -torch.inf, -torch.inf, key)
    key = torch.where(key.isnan(), torch.inf, key)
    if g < G:
        top = key.view(R, G, -1).topk(best, dim=2).values
        if best == 2:
            top = torch.where(top[:, :, 1:] == -torch.inf, torch.cat([top[:, :, :1], torch.zeros_like(top[:, :, 1:])], 2), top)
        total = top.sum(2)
        order = torch.sort(total, dim=1, descending=True, stable=True).indices
        if got is not None:
            edge = total.gather(1, order)[:, g - 1:g]
            near = (total - edge).abs() <= GROUP_TIE
            used = torch.zeros(R, G, dtype=torch.bool).scatter_(1, (got.cpu().long() - S) // (n // G), True)
            # certain groups first, then the undecided ones that the kernel kept, then the other undecided ones
            rank = torch.where(near, torch.where(used, 1.0, 2.0), torch.where(total > edge, 0.0, 3.0))
            # (groups with the same two keys as the last one kept are truly equal: the lower one stays)
            same = (top == top.gather(1, order[:, g - 1:g, None].expand(R, 1, best))).all(2)
            split = (near & ~same).any(1)
            again = torch.sort(rank, dim=1, stable=True).indices
            order = torch.where(split[:, None], again, order)
        live = torch.zeros(R, G, dtype=torch.bool).scatter_(1, order[:, :g], True).repeat_interleave(n // G, 1)
    else:
        live = torch.ones(R, n, dtype=torch.bool)
    # live chapters first, by key descending, ties by position
    pos = torch.sort(key, dim=1, descending=True, stable=True).indices
    pos = torch.take_along_dim(pos, torch.sort((~live.gather(1, pos)).int(), dim=1, stable=True).indices, 1)[:, :k]
    sel = s.gather(1, pos)
    w = scale * (sel / sel.sum(1, keepdim=True).clamp_min(1e-12) if renorm else sel)
    dz = torch.autograd.grad(w, z, dw.cpu().double())[0] if dw is not None else None
    return (pos + S).int(), w.detach(), dz


def run(z, k, S, dev, dw=None, bias=None, **kw):
    from memory_amd import ops
    zd = z.to(dev).requires_grad_(dw is not None)
    idx, w = ops.router_select(zd, k, S, bias=None if bias is None else bias.to(dev), **kw)
    dz = torch.autograd.grad(w, zd, dw.to(dev))[0] if dw is not None else None
    return idx, w.detach(), dz


def compare(z, k, S, dev, seed=0, bias=None, score="softmax", G=1, g=None, best=2, renorm=True, scale=1.0):
    dw = torch.randn(z.shape[0], k, generator=gen(seed + 77))
    idx, w, dz = run(z, k, S, dev, dw, bias, score=score, num_groups=G, top_groups=g, group_best=best, renormalize=renorm,
                     scale=scale)
    ridx, rw, rdz = reference(z, k, S, score, bias, G, g, best, renorm, scale, dw, idx)
    assert idx.dtype == torch.int32 and torch.equal(idx.cpu(), ridx)
    err = ((w.cpu().double() - rw).abs() / rw.abs().amax(1, keepdim=True).clamp_min(1e-30)).max().item()
    big = rdz.abs().amax(1, keepdim=True) + (rw * dw).abs().amax(1, keepdim=True)
    gerr = ((dz.cpu().double() - rdz).abs() / big.clamp_min(1e-30)).max().item()
    print(f"R={z.shape[0]} C={z.shape[1]} k={k} {score} G={G}/{g} weights {err:.2e} gradient {gerr:.2e}", flush=True)
    assert err <= TOL and gerr <= TOL
    assert not dz[:, :S].any()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("G,g,best", [(1, None, 1), (8, 4, 2), (8, 3, 1), (3, 2, 2), (16, 16, 2)])
def test_forms(gpu_device, score, with_bias, renorm, G, g, best):
    S, C = 1, 1 + 48 * 7
    g0 = gen(3)
    z = torch.randn(70, C, generator=g0)
    bias = torch.randn(C, generator=g0) * 0.05 if with_bias else None
    compare(z, 6, S, gpu_device, 1, bias, score, G, g, best, renorm, 2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C,S,k,G,g", [(1, 1, 0, 1, 1, 1), (1, 4097, 1, 64, 8, 4), (3, 4097, 1, 64, 1, 1), (65, 4097, 1, 16, 16, 4),
                                         (200, 4097, 1, 64, 4, 2), (33, 257, 1, 8, 1, 1), (130, 65, 0, 65, 1, 1), (9, 16384, 0, 100, 32, 5),
                                         (2, 16384, 4, 1024, 1, 1), (70, 129, 1, 1, 128, 1), (66, 4609, 1, 64, 64, 20),
                                         (67, 5000, 8, 33, 3, 2), (500, 33, 1, 4, 1, 1), (80, 1025, 1, 300, 2, 1), (77, 64, 2, 20, 31, 10),
                                         (1030, 100, 1, 3, 9, 2), (64, 2049, 1, 128, 1024, 700), (90, 3, 1, 2, 1, 1)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_sizes(gpu_device, R, C, S, k, G, g, score):
    g0 = gen(R + C + k)
    z = torch.randn(R, C, generator=g0) * 0.55
    bias = torch.randn(C, generator=g0) * 0.02
    compare(z, k, S, gpu_device, 2, bias, score, G, g, 2, True, 1.0)
    compare(z, k, S, gpu_device, 3, None, score, G, g, 1, score == "sigmoid", 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("C,S,k,G,g", [(4097, 1, 16, 8, 4), (4097, 1, 64, 1, 1), (4097, 1, 64, 16, 1), (4609, 1, 33, 64, 20),
                                       (257, 1, 8, 1, 1), (65, 1, 64, 1, 1), (301, 1, 20, 3, 1), (4096, 0, 5, 2, 1),
                                       (1366 * 3 + 1, 1, 40, 3, 2), (130, 2, 64, 32, 16), (2049, 1, 64, 4, 1), (17, 1, 16, 1, 1)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_many_rows(gpu_device, C, S, k, G, g, score):
    """More rows than four waves each are taken for: one wave per row, in registers."""
    R = 1030
    g0 = gen(C + k)
    z = torch.randn(R, C, generator=g0) * 0.55
    bias = torch.randn(C, generator=g0) * 0.02
    compare(z, k, S, gpu_device, 2, bias, score, G, g, 2, True, 1.0)
    compare(z, k, S, gpu_device, 3, None, score, G, g, 1, False, 1.0)
    compare(z, k, S, gpu_device, 4, None, score, G, g, 2, True, 2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [5, 300, 1100])
@pytest.mark.parametrize("score,bias_on", [("sigmoid", True), ("softmax", True), ("sigmoid", False), ("softmax", False)])
@pytest.mark.parametrize("G,g", [(1, 1), (8, 4)])
def test_ties_and_near_ties(gpu_device, R, score, bias_on, G, g):
    """Equal logits go to the lower chapter, also where whole groups are equal; keys one float32 step apart, and keys
    that float32 cannot tell apart, are ordered as float64 orders them."""
    C, S, k = 1025, 1, 24
    g0 = gen(9)
    bias = torch.randn(C, generator=g0).mul_(0.01) if bias_on else None
    coarse = (torch.randn(R, C, generator=g0) * 2).round() / 2            # a dozen values
    if bias_on:
        bias = (bias * 100).round() / 100
    compare(coarse, k, S, gpu_device, 1, bias, score, G, g)
    compare(torch.zeros(R, C), k, S, gpu_device, 1, None if bias is None else bias * 0, score, G, g)
    close = 0.25 + torch.randint(-40, 40, (R, C), generator=g0) * 2.0 ** -25     # a few float32 steps
    compare(close, k, S, gpu_device, 1, bias, score, G, g)
    if bias_on:   # scores + bias that agree to 2^-26 .. 2^-40
        b = 0.5 - (torch.sigmoid(close[0].double()) if score == "sigmoid" else torch.softmax(close[0, S:].double(), 0).mean())
        b = b.float().expand(C).contiguous() if b.dim() == 0 else b.float()
        compare(close, k, S, gpu_device, 1, b, score, G, g)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [7, 200, 1100])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_masked_logits(gpu_device, R, score):
    """-inf masks a chapter: rows with fewer live chapters than k, whole groups masked, the lowest finite value."""
    C, S, k = 513, 1, 16
    g0 = gen(4)
    z = torch.randn(R, C, generator=g0)
    z[torch.rand(R, C, generator=g0) < 0.7] = -torch.inf
    z[1, 10:] = -torch.inf                       # nine live chapters
    z[2, S:] = torch.where(torch.arange(C - S) < 256, -torch.inf, z[2, S:])
    z[3, S:] = torch.randn(C - S, generator=g0)
    z[3, 200:] = torch.finfo(torch.float32).min
    z[4, 50:60] = torch.finfo(torch.float32).min
    bias = torch.randn(C, generator=g0) * 0.3
    for b in (None, bias):
        for G, g in ((1, 1), (4, 2)):
            idx, w, dz = run(z, k, S, gpu_device, torch.ones(R, k), b, score=score, num_groups=G, top_groups=g)
            ridx, rw, rdz = reference(z, k, S, score, b, G, g, dw=torch.ones(R, k))
            assert torch.equal(idx.cpu(), ridx)
            assert (w.cpu().double() - rw).abs().max() <= TOL
            assert (dz.cpu().double() - rdz).abs().max() <= TOL


@pytest.mark.gpu
def test_nothing_left_and_not_a_number(gpu_device):
    """A row with every chapter masked names the first k: weight 0 (sigmoid) or NaN (softmax); NaN sorts first; both
    leave the other rows as they are."""
    from memory_amd import ops
    for R in (6, 100, 1100):
        z = torch.randn(R, 300, generator=gen(1)).to(gpu_device)
        for score in ("sigmoid", "softmax"):
            i0, w0 = ops.router_select(z, 5, 1, score=score)
            z1 = z.clone()
            z1[2] = -torch.inf
            z1[4, 77] = torch.nan
            i1, w1 = ops.router_select(z1, 5, 1, score=score)
            rest = [r for r in range(R) if r not in (2, 4)]
            assert torch.equal(i0[rest], i1[rest]) and torch.equal(w0[rest], w1[rest])
            assert i1[2].tolist() == [1, 2, 3, 4, 5]
            assert not w1[2].any() if score == "sigmoid" else w1[2].isnan().all()
            assert i1[4, 0] == 77 and w1[4].isnan().all()
            assert i1[4, 1:].tolist() == [c for c in i0[4].tolist() if c != 77][:4]


@pytest.mark.gpu
def test_layouts_types_and_saturated_scores(gpu_device):
    from memory_amd import ops
    z = torch.randn(90, 512, generator=gen(2))
    wide = z.to(gpu_device)
    i0, w0 = ops.router_select(wide[:, :257].contiguous(), 8, 1, score="sigmoid")
    i1, w1 = ops.router_select(wide[:, :257], 8, 1, score="sigmoid")          # rows of a wider matrix
    assert torch.equal(i0, i1) and torch.equal(w0, w1)
    i1, w1 = ops.router_select(wide[:, :257].t().contiguous().t(), 8, 1, score="sigmoid")
    assert torch.equal(i0, i1) and torch.equal(w0, w1)
    off = torch.empty(90 * 257 + 1, device=gpu_device)[1:].view(90, 257).copy_(wide[:, :257])
    i1, w1 = ops.router_select(off, 8, 1, score="sigmoid")
    assert torch.equal(i0, i1) and torch.equal(w0, w1)
    zb = z[:, :257].bfloat16()
    compare(zb.float(), 8, 1, gpu_device, bias=torch.randn(257, generator=gen(5)) * 0.1, score="sigmoid")
    zg = zb.to(gpu_device).requires_grad_(True)
    idx, w = ops.router_select(zg, 8, 1, score="sigmoid")
    (dz,) = torch.autograd.grad(w.sum() + (w * w).sum(), zg)
    assert dz.dtype == torch.bfloat16 and torch.equal(idx.cpu(), reference(zb.float(), 8, 1, "sigmoid")[0])
    # scores at both ends: 1 - e^-30 and e^-30
    far = torch.cat([z[:, :128] * 4 + 20, z[:, 128:] * 4 - 20], 1)
    compare(far, 8, 0, gpu_device, bias=torch.randn(512, generator=gen(6)) * 1e-3, score="sigmoid")
    compare(far, 8, 0, gpu_device, score="sigmoid", renorm=False)
    compare(far - 20, 8, 0, gpu_device, score="sigmoid", renorm=True)
    compare(far, 8, 0, gpu_device, bias=torch.randn(512, generator=gen(6)), score="softmax", renorm=True)


@pytest.mark.gpu
def test_empty_rows_and_repeats(gpu_device):
    from memory_amd import ops
    z = torch.zeros(0, 33, device=gpu_device, requires_grad=True)
    idx, w = ops.router_select(z, 4, 1)
    assert idx.shape == w.shape == (0, 4)
    assert torch.autograd.grad(w.sum(), z)[0].shape == (0, 33)
    z = torch.randn(3000, 513, generator=gen(8))
    a = run(z, 16, 1, gpu_device, torch.ones(3000, 16), torch.zeros(513), score="sigmoid", num_groups=8, top_groups=3)
    b = run(z, 16, 1, gpu_device, torch.ones(3000, 16), torch.zeros(513), score="sigmoid", num_groups=8, top_groups=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    z[:, ::2] = 0.5      # crowded with equal keys: every row takes the general path
    runs = [run(z, 60, 1, gpu_device, torch.ones(3000, 60), torch.zeros(513), score=s) for s in ("softmax", "sigmoid") * 2]
    assert all(torch.equal(x, y) for i in (0, 1) for x, y in zip(runs[i], runs[i + 2]))


@pytest.mark.gpu
@pytest.mark.parametrize("score,R", [("sigmoid", 16), ("softmax", 300)])
def test_graph_replays(gpu_device, score, R):
    from memory_amd import ops
    C = 1025
    z = torch.randn(R, C, generator=gen(1)).to(gpu_device).requires_grad_(True)
    bias = torch.randn(C, generator=gen(2)).mul_(0.02).to(gpu_device)
    dw = torch.randn(R, 16, generator=gen(3)).to(gpu_device)

    def step():
        idx, w = ops.router_select(z, 16, 1, score=score, bias=bias, num_groups=8, top_groups=4, renormalize=False)
        return idx, w.detach(), torch.autograd.grad(w, z, dw)[0]

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
            z.copy_(torch.randn(R, C, generator=gen(10 + rep)))
        graph.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {rep}"


@pytest.mark.gpu
def test_gradient_against_differences(gpu_device):
    """Central differences of the weights along random directions that leave the selection as it is."""
    from memory_amd import ops
    for score, renorm in (("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)):
        z = torch.randn(4, 65, generator=gen(7))
        dw = torch.randn(4, 5, generator=gen(8))
        idx, w, dz = run(z, 5, 1, gpu_device, dw, score=score, renormalize=renorm)
        v = torch.randn(4, 65, generator=gen(9)) * 2.0 ** -9
        outs = [reference(z.double() + sgn * v.double(), 5, 1, score, renorm=renorm) for sgn in (1, -1)]
        assert all(torch.equal(o[0], idx.cpu()) for o in outs)
        diff = ((outs[0][1] - outs[1][1]) * dw.double()).sum() / 2
        got = (dz.cpu().double() * v.double()).sum()
        # third-order term of the difference: |v|^3 times third derivatives below 1, summed over 4 x 65
        assert abs(diff - got) <= 260 * (8 * 2.0 ** -9) ** 3 + TOL * (dz.cpu().double() * v.double()).abs().sum(), (score, renorm)


@pytest.mark.gpu
@pytest.mark.parametrize("n,C,S", [(0, 33, 1), (5000, 33, 1), (131072, 4097, 1), (70, 16384, 0)])
def test_balance(gpu_device, n, C, S):
    from memory_amd import ops
    idx = torch.randint(S, C, (n,), generator=gen(n + C)).to(torch.int32)
    idx[::5] = S
    bias = torch.randn(C, generator=gen(1))
    want = torch.bincount(idx.long(), minlength=C)
    mean = want[S:].double().mean()
    step = torch.sign(mean - want.double()) * 0.001
    step[:S] = 0
    b = bias.to(gpu_device)
    counts = ops.router_balance_(b, idx.to(gpu_device).view(-1, 1), 0.001, S)
    assert torch.equal(counts.cpu().long(), want)
    assert torch.equal(b.cpu(), bias + step.float())
    stray = torch.tensor([-1, C, S, S], dtype=torch.int32)
    assert ops.router_balance_(b, stray.to(gpu_device), 0.0, S).sum() == 2


def test_refusals():
    from memory_amd import _lib as L
    from memory_amd import ops
    z = torch.zeros(3, 17)
    for bad in (dict(score="relu"), dict(num_groups=3), dict(num_groups=0), dict(num_groups=4, top_groups=5),
                dict(num_groups=4, top_groups=0), dict(group_best=3), dict(bias=torch.zeros(16))):
        with pytest.raises(ValueError):
            ops.router_select(z, 4, 1, **bad)
    for k, S in ((0, 1), (17, 1), (4, 17), (4, -1)):
        with pytest.raises(ValueError):
            ops.router_select(z, k, S)
    with pytest.raises(ValueError):
        ops.router_select(z, 9, 1, num_groups=4, top_groups=2)      # 8 selectable
    with pytest.raises(ValueError):
        ops.router_select(z[0], 4, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.router_select(z, 4, 1)
    with pytest.raises(ValueError, match="float32 vector"):
        ops.router_balance_(torch.zeros(4, dtype=torch.bfloat16), torch.zeros(2), 0.1)
    args = lambda **kw: [{**dict(z=16, ld=17, R=3, C=17, S=1, k=4, score=0, b=None, G=1, g=1, best=1, rn=1, sc=1.0, i=16, w=16,
                                 s=None, st=None, q=None), **kw}[n] for n in ("z", "ld", "R", "C", "S", "k", "score", "b", "G", "g", "best",
                                                                               "rn", "sc", "i", "w", "s", "st", "q")]
    for bad in (dict(C=20000, ld=20000), dict(S=17), dict(score=2), dict(G=5), dict(g=2), dict(best=0), dict(k=1025), dict(ld=16),
                dict(z=None), dict(R=-1)):
        with pytest.raises(ValueError):
            L.call("moc_router_select", *args(**bad))


def test_balance_bias_stays_in_float32():
    from memory_amd.router import ChapterRouter
    r = ChapterRouter(32, 9, 2, balance_bias=True)
    r.balance_bias.copy_(torch.linspace(-0.01, 0.01, 9))
    want = r.balance_bias.clone()
    r = r.to(torch.bfloat16)
    assert r.router.weight.dtype == torch.bfloat16 and r.balance_bias.dtype == torch.float32
    assert torch.equal(r.balance_bias, want) and "balance_bias" in r.state_dict()
    assert torch.equal(r.half().float().balance_bias, want) and r.balance_bias is dict(r.named_buffers())["balance_bias"]
    assert ChapterRouter(32, 9, 2).to(torch.bfloat16).balance_bias is None


def near_cut(R, C, S, best, seed):
    """Peaked softmax rows of two groups, and a bias on the best chapter of the second one: the groups' totals differ
    by 2^-27 .. 2^-40 either way, their scores' sums by about a half.  Two chapters outside either group's best give
    the sum of exponentials its value."""
    g0 = gen(seed)
    n, per = C - S, (C - S) // 2
    z = torch.randn(R, n, generator=g0) - 1
    z[:, per - 2:per] = -20.0                        # the two chapters that set the sum
    z[:, [3, 5]] = 8 + 0.02 * torch.rand(R, 2, generator=g0)
    z[:, [per + 2, per + 7]] = 6.5 + 0.02 * torch.rand(R, 2, generator=g0)
    bias = torch.zeros(C)
    e = z.double().exp()
    pairs = lambda x: x.topk(best, dim=1).values.sum(1)
    # the best of group two with the bias on its chapter: that chapter (and the larger other one)
    two = e[:, per + 2] + (e[:, per + 7] if best == 2 else 0)
    gap = torch.exp2(-27 - 13 * torch.rand(R, generator=g0, dtype=torch.float64)) * torch.where(torch.rand(R, generator=g0) < 0.5, 1.0, -1.0)
    rest = e[:, :per - 2].sum(1) + e[:, per:].sum(1)
    apart = pairs(e[:, :per]) - two
    bias[S + per + 2] = (apart / (rest + 700)).median().float()
    total = apart / (bias[S + per + 2].double() + gap)        # sum of exponentials for which the totals differ by gap
    assert (total - rest > 1).all() and (total - rest < 1500).all()
    z[:, per - 2] = torch.log(total - rest - 2.0 ** -7).float()
    z[:, per - 1] = torch.log(total - rest - z[:, per - 2].double().exp()).float()
    s = torch.softmax(z.double(), 1)
    have = pairs(s[:, :per]) - s[:, per + 2] - (s[:, per + 7] if best == 2 else 0) - bias[S + per + 2].double()
    assert (have.sign() == gap.sign()).all() and (have.abs() > 2.0 ** -42).all() and (have.abs() < 2.0 ** -26).all()
    return torch.cat([torch.zeros(R, S), z], 1), bias


@pytest.mark.gpu
@pytest.mark.parametrize("R", [5, 1100])
@pytest.mark.parametrize("C,k", [(1025, 16), (257, 8), (4097, 64), (1025, 70)])
@pytest.mark.parametrize("best", [1, 2])
def test_softmax_groups_near_the_cut_with_unequal_biases(gpu_device, R, C, k, best):
    """Groups whose totals (scores and biases) differ by less than a float32 sum of exponentials tells apart."""
    z, bias = near_cut(R, C, 1, best, R + C + best)
    compare(z, k, 1, gpu_device, 1, bias, "softmax", 2, 1, best)


def test_near_cut_tells_a_float32_sum_from_an_exact_one():
    """Rows of near_cut change sides where the sum of exponentials is 2^-23 off."""
    z, bias = near_cut(400, 1025, 1, 2, 3)
    zd = z[:, 1:].double()
    sides = []
    for off in (0.0, 2.0 ** -23):
        s = zd.exp() / (zd.exp().sum(1, keepdim=True) * (1 + off)) + bias[1:].double()
        sides.append(s[:, :512].topk(2).values.sum(1) > s[:, 512:].topk(2).values.sum(1))
    assert (sides[0] != sides[1]).float().mean() > 0.2


@pytest.mark.gpu
@pytest.mark.parametrize("R", [9, 1100])
@pytest.mark.parametrize("renorm", [False, True])
def test_sigmoid_gradient_of_saturated_scores(gpu_device, R, renorm):
    """Every element's gradient ds s (1 - s) on its own scale, also where the score rounds to 1 in float32.  The kernel
    forms s (1 - s) from the logit and ds from scores rounded to float32 (2^-24 each), in float64, and rounds the
    result (2^-24): 2^-21 of the terms of ds times s (1 - s), and half a subnormal step."""
    C, S, k = 301, 1, 12
    g0 = gen(31)
    z = torch.randn(R, C, generator=g0)
    at = torch.randperm(C - S, generator=g0)[:k] + S
    z[:, at] = 8 + 50 * torch.rand(R, k, generator=g0)             # s to 1 - e^-58
    z[1] = -60 - 25 * torch.rand(C, generator=g0)                  # and down to e^-85
    dw = torch.randn(R, k, generator=g0)
    idx, w, dz = run(z, k, S, gpu_device, dw, score="sigmoid", renormalize=renorm, scale=1.5)
    ridx, rw, _ = reference(z, k, S, "sigmoid", renorm=renorm, scale=1.5)
    assert torch.equal(idx.cpu(), ridx)
    zs, d = z.double().gather(1, ridx.long()), dw.double()
    s, slope = torch.sigmoid(zs), torch.sigmoid(zs) * torch.sigmoid(-zs)
    if renorm:
        D = s.sum(1, keepdim=True).clamp_min(1e-12)
        shift = torch.where(s.sum(1, keepdim=True) > 1e-12, (d * s).sum(1, keepdim=True) / D, 0.0)
        ds, terms = 1.5 * (d - shift) / D, 1.5 * (d.abs() + (d * s).abs().sum(1, keepdim=True) / D) / D
    else:
        ds, terms = 1.5 * d, 1.5 * d.abs()
    err = (dz.cpu().double().gather(1, ridx.long()) - ds * slope).abs()
    bound = 2.0 ** -21 * terms * slope + 2.0 ** -150
    print(f"worst {(err / bound).max().item():.3f} of the bound", flush=True)
    assert (err <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("R", [9, 1100])
@pytest.mark.parametrize("C,k", [(301, 12), (301, 1), (301, 70), (70, 69)])
def test_softmax_gradient_of_saturated_scores(gpu_device, R, C, k):
    """Scores that are not renormalised, one of them near 1: dz_j = s_j (ds_j (1 - sum of the selected s) + sum_i (ds_j
    - ds_i) s_i), each element on the scale of these terms (TOL, as everywhere in this file)."""
    S = 1
    g0 = gen(33)
    z = torch.randn(R, C, generator=g0)
    z[:, 7] = 2 + 35 * torch.rand(R, generator=g0)
    dw = torch.randn(R, k, generator=g0)
    idx, w, dz = run(z, k, S, gpu_device, dw, score="softmax", renormalize=False, scale=1.5)
    ridx, rw, _ = reference(z, k, S, "softmax", renorm=False, scale=1.5)
    assert torch.equal(idx.cpu(), ridx)
    p = z[:, S:].double()
    p = (p - torch.logsumexp(p, 1, keepdim=True)).exp()
    s, ds = p.gather(1, ridx.long() - S), 1.5 * dw.double()
    left = p.scatter(1, ridx.long() - S, 0.0).sum(1, keepdim=True)
    pairs = ds[:, :, None] - ds[:, None, :]
    want = s * (ds * left + (pairs * s[:, None, :]).sum(2))
    scale = s * (ds.abs() * left + (pairs.abs() * s[:, None, :]).sum(2))
    err = (dz.cpu().double().gather(1, ridx.long()) - want).abs()
    # (float64's own sums of the row leave 2^-48; float32's smallest step)
    bound = TOL * scale + 2.0 ** -48 * s * ds.abs().amax(1, keepdim=True) + 2.0 ** -149
    print(f"worst {(err / bound).max().item():.3f} of the bound", flush=True)
    assert (err <= bound).all()


@pytest.mark.gpu
def test_one_row_of_any_strides(gpu_device):
    """A single row whose row stride says nothing (a transposed column), forward and backward."""
    from memory_amd import ops
    z = torch.randn(1, 257, generator=gen(12)).to(gpu_device)
    dw = torch.randn(1, 8, generator=gen(13)).to(gpu_device)
    column = z.reshape(257, 1).t()
    assert column.stride() == (1, 1)
    for score in ("sigmoid", "softmax"):
        outs = []
        for view in (z, column, z.expand(3, 257)[1:2], z.as_strided((1, 257), (5, 1))):
            leaf = view.detach().requires_grad_(True)
            idx, w = ops.router_select(leaf, 8, 1, score=score, renormalize=False)
            outs.append((idx, w, torch.autograd.grad(w, leaf, dw)[0]))
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(outs[0], ops.router_select(view, 8, 1, score=score, renormalize=False)))
        for o in outs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu_device):
    """A tangent raises, as in the other selection: it is never dropped."""
    import torch.autograd.forward_ad as fwd
    from memory_amd import ops
    z = torch.randn(5, 33, generator=gen(1)).to(gpu_device)
    with fwd.dual_level():
        dual = fwd.make_dual(z, torch.ones_like(z))
        for f in (ops.router_topk, ops.router_select):
            with pytest.raises(NotImplementedError):
                f(dual, 4, 1)
        idx, w = ops.router_select(z, 4, 1)          # (no tangent: as outside)
    assert all(torch.equal(a, b) for a, b in zip((idx, w), ops.router_select(z, 4, 1)))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: ops.router_select(t, 4, 1)[1], (z,), (torch.ones_like(z),))


def test_a_checkpoint_without_a_bias_starts_it_at_zero():
    """Weights loaded over a router whose bias has moved: the bias of a checkpoint that has one, 0 of one that has
    none; a state dict without that router leaves it alone."""
    from memory_amd.checkpoint import MemoryStack
    mem = dict(use_chapters=True, num_chapters=9, num_memory_tokens=9 * 64, top_k_chapters=2, num_shared_chapters=1,
               router_options=dict(balance_bias=True))
    stack = MemoryStack(hidden_dim=64, num_layers=1, num_heads=1, num_kv_heads=None, memory=mem)
    moved = torch.linspace(-1, 1, 9)
    router = next(iter(stack.routers.values()))
    router.balance_bias.copy_(moved)
    whole = {k: v.clone() for k, v in stack.state_dict().items()}
    router.balance_bias.zero_()
    stack.load_reference_state_dict(whole)
    assert torch.equal(router.balance_bias, moved)
    stack.load_reference_state_dict({k: v for k, v in whole.items() if not k.startswith("routers")}, strict=False)
    assert torch.equal(router.balance_bias, moved)
    stack.load_reference_state_dict({k: v for k, v in whole.items() if not k.endswith("balance_bias")})
    assert not router.balance_bias.any()


def test_balance_refuses_more_ids_than_it_counts():
    from memory_amd import _lib as L
    for n in (-1, 1 << 31, 1 << 37):      # (the counts have 32 bits)
        with pytest.raises(ValueError, match="moc_router_balance"):
            L.call("moc_router_balance", 16, n, 9, 1, 0.1, 16, 16, None)
