"""ops.head_norm_rotate and ops.qk_norm_rotate against the same formulas in float64.

Tolerances, derived (u = 2^-24, t = the result's rounding, 2^-8 for bfloat16 and 2^-24 for float32).  A norm's sum of
squares has at most 16 serial and 5 cross-lane roundings, division, root and products 6 more; sine and cosine are off by
2^-23 plus the reduced angle's own rounding (pi u); a rotation adds 3.  So an element is off by at most
48 u max|row| before its store.  In the backward two such sums and the rotation back pass in front of a store:
128 u rstd max|g| (1 + max|xh|), with g the gradient before the norm; a weight's gradient adds (rows + 64) u of its terms'
magnitudes."""

import pytest
import torch

from helpers import gen

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def turned(u, pos, freq, interleaved, back=False):
    """float64 rotation of u (B, L, H, D) by pos (B, L) * freq"""
    if freq is None:
        return u
    R = 2 * freq.shape[0]
    a = pos.double()[..., None, None] * freq.double()
    c, s = a.cos(), a.sin() * (-1 if back else 1)
    if interleaved:
        x, y = u[..., 0:R:2], u[..., 1:R:2]
        rot = torch.stack([x * c - y * s, y * c + x * s], -1).flatten(-2)
    else:
        x, y = u[..., :R // 2], u[..., R // 2:R]
        rot = torch.cat([x * c - y * s, y * c + x * s], -1)
    return torch.cat([rot, u[..., R:]], -1)


def reference(x, w, eps, norm, pos, freq, interleaved, dy=None):
    t = 2.0 ** -8 if x.dtype == BF else 2.0 ** -24
    xd = x.detach().double()
    rs = (xd.square().mean(-1, keepdim=True) + eps).rsqrt() if norm else torch.ones_like(xd[..., :1])
    xh = xd * rs
    wd = torch.ones((), dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    u = xh * wd
    y = turned(u, pos, freq, interleaved)
    by = t * y.abs() + 48 * U * u.abs().amax(-1, keepdim=True)
    if dy is None:
        return y, by
    du = turned(dy.double(), pos, freq, interleaved, back=True)
    g = du * wd
    dx = rs * (g - xh * (g * xh).mean(-1, keepdim=True)) if norm else g
    gm = (dy.double().abs().amax(-1, keepdim=True) * 1.5) * wd.abs().max()      # (a turned pair grows by at most root 2)
    bx = t * dx.abs() + 128 * U * rs * gm * (1 + (xh.abs().amax(-1, keepdim=True) if norm else 0))
    if w is None:
        return (y, dx), (by, bx)
    terms = du * xh
    over = (0, 1) if w.dim() == 2 else (0, 1, 2)
    n = terms.numel() // terms.shape[-1]
    mag = (dy.double().abs().amax(-1, keepdim=True) * 1.5) * xh.abs()
    return (y, dx, terms.sum(over)), (by, bx, (n + 64 + 48) * U * mag.sum(over) + U * terms.sum(over).abs())


def close(got, ref, bound, what):
    assert torch.isfinite(got).all(), what
    over = ((got.double() - ref).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 1e-30, f"{what}: {over:.3e} above the bound (largest {bound.max().item():.3e})"


def data(dev, dt, B, L, H, D, weight, seed=0):
    g = gen(seed)
    x = torch.randn(B, L, H, D, generator=g).to(dt).to(dev).requires_grad_(True)
    w = None
    if weight != "none":
        w = (1 + 0.1 * torch.randn(*((H, D) if weight == "head" else (D,)), generator=g)).to(dev).requires_grad_(True)
    return x, w, torch.randn(B, L, H, D, generator=g).to(dt).to(dev)


CASES = [  # B, L, H, D, R, interleaved, weight, norm
    (1, 1, 1, 64, 64, False, "shared", True), (2, 7, 12, 64, 64, False, "shared", True),
    (3, 5, 4, 128, 64, True, "head", True), (2, 9, 32, 128, 128, False, "head", True), (1, 33, 3, 96, 32, False, "shared", True),
    (2, 5, 5, 80, 80, True, "none", True), (2, 4, 3, 30, 14, False, "head", True), (1, 6, 2, 2, 2, True, "shared", True),
    (2, 3, 2, 512, 512, False, "shared", True), (1, 3, 3, 510, 256, True, "head", True), (2, 5, 4, 64, 32, False, "none", False),
    (2, 5, 4, 40, 24, False, "none", False), (2, 5, 4, 64, 0, False, "shared", True), (1, 700, 2, 64, 64, True, "shared", True),
    (2, 3, 70, 64, 48, False, "head", True), (1, 2, 9, 16, 10, True, "head", True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(gpu_device, case, dt):
    from memory_amd import ops
    B, L, H, D, R, inter, weight, norm = case
    x, w, dy = data(gpu_device, dt, B, L, H, D, weight)
    freq = ops.rope_frequencies(R, 10000.0, gpu_device) if R else None
    pos = (torch.arange(L) + 11)[None].expand(B, L).to(gpu_device)
    kw = dict(norm=norm, inv_freq=freq, interleaved=inter)
    if R:
        kw["positions"] = pos
    y = ops.head_norm_rotate(x, w, **kw)
    leaves = [x] if w is None else [x, w]
    grads = torch.autograd.grad(y, leaves, dy)
    ref, bound = reference(x, w, 1e-6, norm, pos, freq, inter, dy)
    for name, a, b, c in zip(("y", "dx", "dw"), (y.detach(), *grads), ref, bound):
        close(a, b, c, name)
    with torch.no_grad():
        assert torch.equal(y.detach(), ops.head_norm_rotate(x, w, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
def test_both_in_one(gpu_device, dt):
    """qk_norm_rotate is head_norm_rotate of each, with other rows, heads, weights and positions; a gradient of one
    alone leaves the other's parameters out."""
    from memory_amd import ops
    q, wq, dq = data(gpu_device, dt, 2, 37, 12, 64, "shared")
    k, wk, dk = data(gpu_device, dt, 2, 101, 3, 64, "head", seed=1)
    freq = ops.rope_frequencies(64, 500.0, gpu_device)
    pq = torch.randint(0, 5000, (2, 37), generator=gen(2)).to(gpu_device)
    pk = torch.randint(-300, 300, (101,), generator=gen(3), dtype=torch.int32).to(gpu_device)
    a, b = ops.qk_norm_rotate(q, k, wq, wk, q_positions=pq, k_positions=pk, inv_freq=freq)
    got = torch.autograd.grad([a, b], [q, k, wq, wk], [dq, dk])
    a1, b1 = ops.head_norm_rotate(q, wq, positions=pq, inv_freq=freq), ops.head_norm_rotate(k, wk, positions=pk, inv_freq=freq)
    assert torch.equal(a, a1) and torch.equal(b, b1)
    ref, bound = reference(q, wq, 1e-6, True, pq, freq, False, dq)
    for name, i, x in (("dq", 1, got[0]), ("dwq", 2, got[2])):
        close(x, ref[i], bound[i], name)
    ref, bound = reference(k, wk, 1e-6, True, pk[None].expand(2, 101), freq, False, dk)
    for name, i, x in (("dk", 1, got[1]), ("dwk", 2, got[3])):
        close(x, ref[i], bound[i], name)
    a, b = ops.qk_norm_rotate(q, k, wq, wk, q_positions=pq, k_positions=pk, inv_freq=freq)
    one = torch.autograd.grad(a, [q, k, wq, wk], dq, allow_unused=True)
    assert one[1] is None and one[3] is None
    ref, bound = reference(q, wq, 1e-6, True, pq, freq, False, dq)
    close(one[0], ref[1], bound[1], "dq")
    close(one[2], ref[2], bound[2], "dwq")


@pytest.mark.gpu
@pytest.mark.parametrize("start", [0, 10 ** 6, 2 ** 31 + 7, -(10 ** 6)])
def test_far_positions(gpu_device, start):
    """Angles of far positions, reduced in float64: the position times a frequency is rounded by 2^-53, so at 2^31
    turns the angle is off by some 5e-7; |y| gets that much more."""
    from memory_amd import ops
    x = torch.randn(1, 40, 2, 64, generator=gen(4)).to(gpu_device)
    pos = (start + torch.arange(40)).to(gpu_device)
    freq = ops.rope_frequencies(64, 10000.0, gpu_device)
    y = ops.head_norm_rotate(x, norm=False, positions=pos, inv_freq=freq)
    ref, bound = reference(x, None, 0, False, pos[None], freq, False)
    close(y, ref, bound + 4 * abs(start) * 2.0 ** -53 * x.double().abs().amax(-1, keepdim=True), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
def test_strides(gpu_device, dt):
    """Slices of a fused projection, heads before rows, a last dim that is not contiguous, odd storage offsets,
    expanded rows; upstream gradients alike."""
    from memory_amd import ops
    g = gen(5)
    fused = torch.randn(2, 6, 10, 64, generator=g).to(dt).to(gpu_device)
    flat = torch.randn(2 * 6 * 4 * 64 + 3, generator=g).to(dt).to(gpu_device)
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(gpu_device)
    freq = ops.rope_frequencies(32, 10000.0, gpu_device)
    pos = torch.arange(6, device=gpu_device)[None].expand(2, 6)
    big = torch.randn(2, 4, 6, 128, generator=g).to(dt).to(gpu_device)
    for x in (fused[:, :, 3:7], fused.transpose(1, 2)[:, 2:6].transpose(1, 2), flat[3:].view(2, 6, 4, 64),
              big[..., ::2].transpose(1, 2), fused[:1, :, :4].expand(2, 6, 4, 64)):
        x = x.detach().requires_grad_(True)
        for dy in (fused[:, :, 6:10], flat[1:-2].view(2, 6, 4, 64), big[..., ::2].transpose(1, 2), fused[:, :, :1].expand(2, 6, 4, 64)):
            y = ops.head_norm_rotate(x, w, positions=pos, inv_freq=freq)
            (dx,) = torch.autograd.grad(y, x, dy)
            ref, bound = reference(x, w, 1e-6, True, pos, freq, False, dy)
            close(y.detach(), ref[0], bound[0], "y")
            close(dx, ref[1], bound[1], "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("off,step", [(0, 0), (2, 0), (1, 0), (2, 6), (3, 5)])
@pytest.mark.parametrize("D,R,inter", [(64, 20, False), (128, 72, False), (96, 56, False), (64, 22, False), (128, 40, True), (48, 2, True),
                                       (256, 4, False), (64, 64, False)])
def test_parts_and_bases(gpu_device, D, R, inter, off, step, dt):
    """Rotated parts that end inside a run of eight, and rows that start at 2, 4, 6 bytes past a 16-byte piece."""
    from memory_amd import ops
    B, L, H = 2, 19, 3
    g = gen(D + R + off)

    def rows():
        n = B * L * H * (D + step)
        flat = torch.full((n + off,), float("nan"), dtype=dt, device=gpu_device)
        x = flat[off:].view(B, L, H, D + step)[..., :D]
        x.copy_(torch.randn(B, L, H, D, generator=g))
        return x
    x, dy = rows().requires_grad_(True), rows()
    w = (1 + 0.1 * torch.randn(H, D, generator=g)).to(gpu_device).requires_grad_(True)
    freq = ops.rope_frequencies(R, 1000.0, gpu_device)
    pos = (torch.arange(L) * 3 + 1)[None].expand(B, L).to(gpu_device)
    y = ops.head_norm_rotate(x, w, positions=pos, inv_freq=freq, interleaved=inter)
    got = (y.detach(), *torch.autograd.grad(y, [x, w], dy))
    ref, bound = reference(x, w, 1e-6, True, pos, freq, inter, dy)
    for name, a, b, c in zip(("y", "dx", "dw"), got, ref, bound):
        close(a, b, c, name)


@pytest.mark.gpu
def test_gradient_against_differences(gpu_device):
    from memory_amd import ops
    x, w, dy = data(gpu_device, F32, 2, 9, 3, 64, "head", seed=6)
    freq = ops.rope_frequencies(48, 100.0, gpu_device)
    pos = torch.arange(9, device=gpu_device)[None].expand(2, 9)
    grads = torch.autograd.grad(ops.head_norm_rotate(x, w, inv_freq=freq), [x, w], dy)
    _, bound = reference(x, w, 1e-6, True, pos, freq, False, dy)
    h = 1e-5

    def value(xd, wd):
        u = xd * (xd.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wd
        return (turned(u, pos, freq, False) * dy.double()).sum()

    for i in range(2):
        d = torch.randn((x, w)[i].shape, generator=gen(7 + i)).to(gpu_device).double()
        args = [[x.detach().double(), w.detach().double()] for _ in range(2)]
        args[0][i] = args[0][i] + h * d
        args[1][i] = args[1][i] - h * d
        diff = ((value(*args[0]) - value(*args[1])) / (2 * h)).item()
        got = (grads[i].double() * d).sum().item()
        assert abs(got - diff) <= (bound[1 + i] * d.abs()).sum().item() + 1e-7 * (grads[i].double() * d).abs().sum().item()


@pytest.mark.gpu
def test_edge_rows(gpu_device):
    """Rows of zeros (eps alone), no rows, one set empty, float16, float32 frequencies."""
    from memory_amd import ops
    freq = ops.rope_frequencies(64, 10000.0, gpu_device)
    x = torch.zeros(1, 3, 2, 64, device=gpu_device, requires_grad=True)
    y = ops.head_norm_rotate(x, inv_freq=freq)
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert (y == 0).all() and torch.isfinite(dx).all()
    k = torch.randn(2, 0, 2, 64, device=gpu_device, requires_grad=True)
    q = torch.randn(2, 5, 4, 64, device=gpu_device, requires_grad=True)
    w = torch.ones(64, device=gpu_device, requires_grad=True)
    a, b = ops.qk_norm_rotate(q, k, w, w, inv_freq=freq)
    gq, gk, gw = torch.autograd.grad([a, b], [q, k, w], [torch.ones_like(a), torch.ones_like(b)])
    assert b.shape == k.shape and gk.shape == k.shape and torch.isfinite(gw).all() and gq.abs().max() > 0
    a, b = ops.qk_norm_rotate(k, k, w, w)
    (gw,) = torch.autograd.grad([a, b], [w], [torch.ones_like(a), torch.ones_like(b)])
    assert (gw == 0).all()
    with torch.no_grad():
        assert ops.head_norm_rotate(k, w).shape == k.shape
        h = torch.randn(1, 4, 2, 64, generator=gen(8)).half().to(gpu_device)
        y = ops.head_norm_rotate(h, w, inv_freq=freq.float())
        assert y.dtype == torch.float16
        ref, _ = reference(h.float(), w, 1e-6, True, torch.arange(4, device=gpu_device)[None], freq.float(), False)
        assert ((y.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 1e-5).all()


@pytest.mark.gpu
def test_captured(gpu_device):
    from memory_amd import ops
    q, wq, dq = data(gpu_device, BF, 4, 33, 12, 64, "shared", seed=9)
    k, wk, dk = data(gpu_device, BF, 4, 60, 3, 64, "head", seed=10)
    pos = torch.arange(33, device=gpu_device)
    freq = ops.rope_frequencies(64, 10000.0, gpu_device)

    def step():
        a, b = ops.qk_norm_rotate(q, k, wq, wk, q_positions=pos, inv_freq=freq)
        return (a.detach(), b.detach(), *torch.autograd.grad([a, b], [q, k, wq, wk], [dq, dk]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=gen(20 + rep)).to(BF))
            pos.add_(100)
        graph.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {rep}"


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu_device):
    """2.3 G elements: the last token's rows, and their gradient."""
    from memory_amd import ops
    x = torch.zeros(1, 70001, 256, 128, device=gpu_device, dtype=BF)
    g = torch.Generator(device=gpu_device).manual_seed(11)
    x[:, -1].normal_(generator=g)
    dy = torch.zeros_like(x)
    dy[:, -1].normal_(generator=g)
    x.requires_grad_(True)
    w = torch.ones(128, device=gpu_device, requires_grad=True)
    freq = ops.rope_frequencies(128, 10000.0, gpu_device)
    y = ops.head_norm_rotate(x, w, inv_freq=freq)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    pos = torch.tensor([[70000]], device=gpu_device)
    ref, bound = reference(x[:, -1:].detach(), w, 1e-6, True, pos, freq, False, dy[:, -1:])
    close(y[:, -1:].detach(), ref[0], bound[0], "y")
    close(dx[:, -1:], ref[1], bound[1], "dx")
    close(dw, ref[2], bound[2], "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("D,R", [(128, 72), (128, 64), (64, 20), (50, 6), (64, 2), (62, 62), (64, 34)])
def test_dims_that_do_not_turn_keep_their_values(gpu_device, D, R, pairs, dt):
    """Infinities and NaN behind the rotated dims stay in their elements, forward and (without a norm) backward; inside
    them they reach their own pair and no other."""
    from memory_amd import ops
    g = gen(60)
    x, dy = (torch.randn(2, 5, 4, D, generator=g).to(dt) for _ in range(2))
    for i, bad in enumerate((float("inf"), float("-inf"), float("nan"))):
        x[:, i, :, R + i::5] = bad
        dy[:, i, :, R + i + 1::5] = bad
    x, dy = x.to(gpu_device).requires_grad_(True), dy.to(gpu_device)
    kw = dict(norm=False, inv_freq=ops.rope_frequencies(R, 10000.0, gpu_device), interleaved=pairs)
    y = ops.head_norm_rotate(x, **kw)
    (dx,) = torch.autograd.grad(y, x, dy)
    for got, want in ((y.detach(), x.detach()), (dx, dy)):
        # NaN compares as one value; the rest of the elements to the bit
        assert torch.equal(got[..., R:].nan_to_num(7.0, 8.0, 9.0), want[..., R:].nan_to_num(7.0, 8.0, 9.0))
        assert torch.isfinite(got[..., :R]).all()
    x = torch.randn(1, 1, 1, D, generator=g).to(dt)
    other = torch.ones(D, dtype=torch.bool)
    for p in {0, R // 2 - 1}:
        z = x.clone()
        a, b = (2 * p, 2 * p + 1) if pairs else (p, R // 2 + p)
        z[..., a] = float("nan")
        keep = other.clone()
        keep[[a, b]] = False
        y = ops.head_norm_rotate(z.to(gpu_device), positions=torch.tensor([3], device=gpu_device), **kw).cpu()
        assert torch.isnan(y[..., ~keep]).all() and torch.isfinite(y[..., keep]).all()
