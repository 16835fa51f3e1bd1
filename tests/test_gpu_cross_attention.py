"""ops.cross_attention against the same formulas in float64, element by element, and MemoryCrossAttention over states
of any length.

Tolerances, derived (u = 2^-24, r = the rounding of the products' operands: 2^-8 for bfloat16, 2^-16 where it takes two
pieces (at most 128 keys or rows of a kv head), 0 for float32; t = the rounding of the result, 2^-8 or 2^-24):
  a logit's error is at most e = (D + 8) u max_j sum_d |q_d k_jd| scale, a probability's 2 e + (N + 64) u relative (the row
  sum has at most N + 64 roundings; 2^-22 for exp2 and log2 is among the 64 u)
  result       t |o| + (2 r + 4 e + 2 (N + 64) u) sum_j p_j |v_j|    (the factor 2: numerator and denominator)
  delta        sum_d |dO_d| (error of o_d before its rounding, plus 2^-16 |o_d| for bfloat16's low piece)
  dS_ij        r |dS_ij| + p_ij ((2 e + (N + 64) u) |dP_ij - delta_i| + (D + 8) u sum_d |dO_d v_jd| + error of delta_i)
  dq, dk       t |.| + scale times the sums of those against |k_j|, |q_i|, with (terms + 64) u of the terms' magnitudes
  dv           t |.| + sum_i (r + 2 e + (N + rows + 128) u) p_ij |dO_i|"""

import pytest
import torch

from helpers import gen

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def reference(q, k, v, live=None, do=None, scale=None):
    """(out, bound) or with do (out, dq, dk, dv and their bounds), float64, one (sequence, head) after the other."""
    dt = q.dtype
    B, L, H, D = q.shape
    N, HK = k.shape[1], k.shape[2]
    G = H // HK
    scale = D ** -0.5 if scale is None else scale
    few = N <= 128 or L * G <= 128
    r = 0.0 if dt == F32 else 2.0 ** -16 if few else 2.0 ** -8
    t = 2.0 ** -24 if dt == F32 else 2.0 ** -8
    qd, kd, vd = q.detach().double(), k.detach().double(), v.detach().double()
    z = lambda x: torch.zeros(x.shape, device=x.device, dtype=torch.float64)
    out, bo = z(q), z(q)
    dq, dk, dv, bq, bk, bv = z(q), z(k), z(k), z(q), z(k), z(k)
    for b in range(B):
        rows = torch.arange(N, device=q.device) if live is None else live[b].nonzero().view(-1)
        if rows.numel() == 0:
            continue
        for h in range(H):
            Q, K, V = qd[b, :, h], kd[b, rows, h // G], vd[b, rows, h // G]
            p = torch.softmax(Q @ K.t().contiguous() * scale, 1)
            e = (D + 8) * U * (Q.abs() @ K.abs().t().contiguous()).amax(1, keepdim=True) * scale
            ep = 2 * e + (N + 64) * U
            o = p @ V
            raw = (2 * r + 2 * ep) * (p @ V.abs())
            out[b, :, h], bo[b, :, h] = o, t * o.abs() + raw
            if do is None:
                continue
            dO = do[b, :, h].double()
            dP = dO @ V.t().contiguous()
            delta = (dO * o).sum(1, keepdim=True)
            edelta = (dO.abs() * (raw + (2.0 ** -16 if dt == BF else t) * o.abs())).sum(1, keepdim=True)
            edelta = edelta + (D + 8) * U * (dO * o).abs().sum(1, keepdim=True)
            dS = p * (dP - delta)
            eS = r * dS.abs() + p * (ep * (dP - delta).abs() + (D + 8) * U * (dO.abs() @ V.abs().t().contiguous()) + edelta)
            dq[b, :, h] = scale * dS @ K
            bq[b, :, h] = t * dq[b, :, h].abs() + scale * (eS + (N + 64) * U * dS.abs()) @ K.abs()
            dSt = dS.t().contiguous()
            dk[b, rows, h // G] += scale * dSt @ Q
            bk[b, rows, h // G] += scale * (eS + (G * L + 64) * U * dS.abs()).t().contiguous() @ Q.abs()
            dv[b, rows, h // G] += p.t().contiguous() @ dO
            bv[b, rows, h // G] += ((r + ep + (G * L + 64) * U) * p).t().contiguous() @ dO.abs()
    if do is None:
        return out, bo
    return (out, dq, dk, dv), (bo, bq, bk + t * dk.abs(), bv + t * dv.abs())


def close(got, ref, bound, what):
    assert torch.isfinite(got).all(), what
    over = ((got.double() - ref).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 1e-30, f"{what}: {over:.3e} above the bound (largest {bound.max().item():.3e})"


def inputs(B, L, N, H, HK, D, dt, dev, seed=0, train=False):
    g = gen(seed)
    q, k, v, do = (torch.randn(*s, generator=g).to(dt).to(dev) for s in
                   ((B, L, H, D), (B, N, HK, D), (B, N, HK, D), (B, L, H, D)))
    if train:
        q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    return q, k, v, do


def check(q, k, v, do, live=None, scale=None, **kw):
    from memory_amd import ops
    if do is None:
        with torch.no_grad():
            o = ops.cross_attention(q, k, v, softmax_scale=scale, **kw)
        ref, bound = reference(q, k, v, live, None, scale)
        close(o, ref, bound, "out")
        return o
    o = ops.cross_attention(q, k, v, softmax_scale=scale, **kw)
    grads = torch.autograd.grad(o, [q, k, v], do)
    ref, bound = reference(q, k, v, live, do, scale)
    for name, x, a, bnd in zip(("out", "dq", "dk", "dv"), (o.detach(), *grads), ref, bound):
        close(x, a, bnd, name)
    return (o.detach(), *grads)


SHAPES = [(1, 1, 1, 1, 1, 64), (2, 3, 5, 4, 2, 64), (1, 16, 64, 2, 2, 128), (2, 17, 65, 4, 1, 64), (1, 129, 63, 2, 2, 64),
          (2, 128, 130, 3, 3, 128), (1, 300, 333, 4, 2, 64), (1, 131, 257, 8, 1, 128), (3, 40, 700, 6, 2, 64),
          (1, 5, 1999, 2, 1, 64), (1, 260, 129, 1, 1, 128), (1, 2100, 5, 8, 1, 64), (1, 700, 200, 4, 1, 128),
          (2, 50, 60, 30, 2, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_training(gpu_device, shape, dt):
    check(*inputs(*shape, dt, gpu_device, train=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES + [(2, 1, 900, 12, 12, 64), (5, 4, 130, 16, 4, 128), (1, 1, 5000, 16, 1, 128)])
def test_forward(gpu_device, shape, dt):
    q, k, v, _ = inputs(*shape, dt, gpu_device, seed=1)
    check(q, k, v, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L", [1, 3, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(gpu_device, L, D, dt):
    """Ragged lengths, a sequence without keys, one with a single key; values past N and below 0 are clamped."""
    N = 203
    lens = torch.tensor([0, 1, 64, 65, 203, 500, -3, 130], device=gpu_device, dtype=torch.int32)
    live = torch.arange(N, device=gpu_device)[None] < lens[:, None]
    q, k, v, do = inputs(8, L, N, 4, 2, D, dt, gpu_device, seed=2, train=True)
    o, dq, dk, dv = check(q, k, v, do, live, kv_lengths=lens)
    for x in (o, dq, dk, dv):
        assert (x[0] == 0).all() and (x[6] == 0).all()
    assert (dk[~live] == 0).all() and (dv[~live] == 0).all()
    o64 = check(q.detach(), k.detach(), v.detach(), None, live, kv_lengths=lens.long())
    assert (o64[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L", [1, 150])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), "lowest"])
def test_mask_hides_what_it_masks(gpu_device, L, D, dt, bad):
    """Keys that do not count hold NaN, infinities or the type's lowest value; whole tiles, single keys and a whole
    sequence are masked, with lengths on top."""
    B, N = 4, 300
    q, k, v, do = inputs(B, L, N, 4, 2, D, dt, gpu_device, seed=3)
    mask = torch.rand(B, N, generator=gen(4)) > 0.4
    mask[0, 64:192] = False
    mask[1] = False
    mask[2] = False
    mask[2, 299] = True
    mask = mask.to(gpu_device)
    lens = torch.tensor([300, 300, 300, 170], device=gpu_device, dtype=torch.int32)
    live = mask & (torch.arange(N, device=gpu_device)[None] < lens[:, None])
    bad = torch.finfo(dt).min if bad == "lowest" else bad
    k[~live] = bad
    v[~live] = bad
    k, v = torch.where(live[..., None, None], k, bad), torch.where(live[..., None, None], v, bad)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o, dq, dk, dv = check(q, k, v, do, live, kv_lengths=lens, key_mask=mask)
    assert (o[1] == 0).all() and (dq[1] == 0).all() and (dk[~live] == 0).all() and (dv[~live] == 0).all()
    check(q.detach(), k.detach(), v.detach(), None, live, kv_lengths=lens, key_mask=mask)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L", [2, 200])
def test_large_logits(gpu_device, L, dt):
    """Logits in the hundreds of both signs: one key takes a row, or all are far below zero."""
    q, k, v, do = inputs(2, L, 150, 2, 1, 64, dt, gpu_device, seed=5)
    q, k = q * 6, k * 6
    k[1] = -q[1, :1, :1].abs()          # row 0 of sequence 1 has negative logits only
    check(*(x.detach().requires_grad_(True) for x in (q, k, v)), do)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L", [1, 90])
def test_strides(gpu_device, L, dt):
    """Slices of fused projections, heads before rows, a shared memory, an expanded batch, unaligned storage."""
    from memory_amd import ops
    g = gen(6)
    B, N, H, HK, D = 2, 77, 4, 2, 64
    qkv = torch.randn(B, L, H + 2, D, generator=g).to(dt).to(gpu_device)
    kv = torch.randn(B, 2, HK, N, D, generator=g).to(dt).to(gpu_device)
    flat = torch.randn(B * N * HK * D + 1, generator=g).to(dt).to(gpu_device)
    q = qkv[:, :, 1:H + 1]
    k, v = kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
    odd = flat[1:].view(B, N, HK, D)
    do = torch.randn(B, H, L, D, generator=g).to(dt).to(gpu_device).transpose(1, 2)
    shared = k[0]
    for a, b, c in ((q, k, v), (q, odd, v), (q.transpose(1, 2).contiguous().transpose(1, 2), k, odd),
                    (q[..., ::2].repeat(1, 1, 1, 2)[..., :D], k, v), (q[:1].expand(B, L, H, D), k, v)):
        check(*(x.detach().requires_grad_(True) for x in (a, b, c)), do)
        check(a, b, c, None)
    one = shared.detach().clone().requires_grad_(True)
    qq = q.detach().requires_grad_(True)
    o = ops.cross_attention(qq, one, one)
    dq, dm = torch.autograd.grad(o, [qq, one], do)
    e = one.detach().expand(B, N, HK, D)
    ref, bound = reference(qq, e, e, None, do)
    close(o.detach(), ref[0], bound[0], "out")
    close(dq, ref[1], bound[1], "dq")
    # (dk and dv of each sequence are rounded to the type, added over the batch and then to each other there)
    t = 2.0 ** -8 if dt == BF else 2.0 ** -24
    close(dm, (ref[2] + ref[3]).sum(0), (bound[2] + bound[3] + 3 * t * (ref[2].abs() + ref[3].abs())).sum(0), "dm")


@pytest.mark.gpu
def test_empty_and_float16(gpu_device):
    from memory_amd import ops
    for B, L, N in ((0, 3, 5), (2, 0, 5), (2, 3, 0)):
        q, k, v, do = inputs(B, L, N, 2, 2, 64, BF, gpu_device, train=True)
        mask = torch.ones(B, N, dtype=torch.bool, device=gpu_device)
        for kw in ({}, dict(key_mask=mask), dict(kv_lengths=torch.zeros(B, dtype=torch.int64, device=gpu_device))):
            o = ops.cross_attention(q, k, v, **kw)
            assert o.shape == q.shape and (o == 0).all()
            assert all((x == 0).all() for x in torch.autograd.grad(o, [q, k, v], do))
    q, k, v, _ = inputs(2, 9, 33, 2, 1, 64, torch.float16, gpu_device)
    o = ops.cross_attention(q, k, v)
    assert o.dtype == torch.float16
    ref, _ = reference(q.float(), k.float(), v.float())
    assert ((o.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gradient_against_differences(gpu_device, D):
    """The kernels' gradient of sum(out * w) along a direction against a central difference of the float64 formula
    (h = 1e-4: truncation and rounding of the quotient below 1e-7 of its terms)."""
    from memory_amd import ops
    q, k, v, w = inputs(2, 30, 75, 4, 2, D, F32, gpu_device, seed=7, train=True)
    lens = torch.tensor([75, 40], device=gpu_device, dtype=torch.int32)
    live = torch.arange(75, device=gpu_device)[None] < lens[:, None]
    grads = torch.autograd.grad(ops.cross_attention(q, k, v, kv_lengths=lens), [q, k, v], w)
    h = 1e-4
    for i, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, generator=gen(8 + i)).to(gpu_device).double()
        val = []
        for s in (h, -h):
            y = [t.detach().double() for t in (q, k, v)]
            y[i] = y[i] + s * d
            val.append((formula(*y, live) * w.double()).sum())
        diff = ((val[0] - val[1]) / (2 * h)).item()
        got = (grads[i].double() * d).sum().item()
        _, bounds = reference(q, k, v, live, w)
        assert abs(got - diff) <= (bounds[1 + i] * d.abs()).sum().item() + 1e-6 * (grads[i].double() * d).abs().sum().item()


def formula(q, k, v, live):
    G = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    s = (q[:, :, None] * k[:, None]).sum(-1) * q.shape[-1] ** -0.5          # (B, L, N, H)
    p = torch.softmax(s.masked_fill(~live[:, None, :, None], float("-inf")), 2)
    return (p[..., None] * v[:, None]).sum(2)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 200, 333, 4, 2, 64), (1, 30, 3000, 8, 2, 128), (2, 1, 900, 4, 4, 64)])
def test_streams_and_repeats(gpu_device, shape):
    """The same bits again, and on another stream."""
    from memory_amd import ops
    q, k, v, do = inputs(*shape, BF, gpu_device, seed=9, train=True)

    def step():
        o = ops.cross_attention(q, k, v)
        return (o.detach(), *torch.autograd.grad(o, [q, k, v], do))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, other, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 33])
def test_captured(gpu_device, L):
    """A captured step replayed on new inputs and lengths, with eager work in between, gives the eager bits."""
    from memory_amd import ops
    q, k, v, do = inputs(3, L, 700, 4, 2, 64, BF, gpu_device, seed=10, train=True)
    lens = torch.tensor([700, 3, 0], device=gpu_device, dtype=torch.int32)
    mask = torch.ones(3, 700, dtype=torch.bool, device=gpu_device)

    def step():
        with torch.no_grad():
            a = ops.cross_attention(q, k, v, kv_lengths=lens)
        o = ops.cross_attention(q, k, v, kv_lengths=lens, key_mask=mask)
        return (a, o.detach(), *torch.autograd.grad(o, [q, k, v], do))

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
            k.copy_(torch.randn(k.shape, generator=gen(20 + rep)).to(BF))
            lens.copy_(torch.tensor([(37 * rep) % 700, 700 - rep, rep], dtype=torch.int32))
            mask.copy_(torch.rand(3, 700, generator=gen(30 + rep)) > 0.3)
        graph.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {rep}"


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu_device):
    """K and V of 2.4 G elements: the last sequence's and heads' rows, forward of one token and of many."""
    from memory_amd import ops
    N, HK, D = 300001, 32, 128
    g = torch.Generator(device=gpu_device).manual_seed(11)
    k = torch.empty(2, N, HK, D, device=gpu_device, dtype=BF)
    k[1, :, 31].normal_(generator=g)
    v = torch.empty(2, N, HK, D, device=gpu_device, dtype=BF)
    v[1, :, 31].normal_(generator=g)
    lens = torch.tensor([0, N], device=gpu_device, dtype=torch.int32)
    for L in (1, 70):
        q = torch.randn(2, L, HK, D, generator=g, device=gpu_device).to(BF)
        with torch.no_grad():
            o = ops.cross_attention(q, k, v, kv_lengths=lens)
        ref, bound = reference(q[1:, :, 31:], k[1:, :, 31:], v[1:, :, 31:])
        close(o[1:, :, 31:], ref, bound + 2.0 ** -7 * 0, f"{L} rows")
        assert (o[0] == 0).all()


@pytest.mark.gpu
def test_second_derivatives_are_refused(gpu_device):
    from memory_amd import ops
    q, k, v, _ = inputs(1, 4, 9, 2, 1, 64, F32, gpu_device, train=True)
    (g,) = torch.autograd.grad(ops.cross_attention(q, k, v).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_partial_gradients(gpu_device):
    """Only some of q, k and v trained: their gradients are those of the whole."""
    from memory_amd import ops
    q, k, v, do = inputs(2, 50, 99, 4, 2, 64, BF, gpu_device, seed=12)
    full = {}
    for names in ("qkv", "q", "k", "v", "kv"):
        t = {n: x.detach().requires_grad_(n in names) for n, x in zip("qkv", (q, k, v))}
        got = torch.autograd.grad(ops.cross_attention(t["q"], t["k"], t["v"]), [t[n] for n in names], do)
        if names == "qkv":
            full = dict(zip(names, got))
        assert all(torch.equal(full[n], x) for n, x in zip(names, got))


# ------------------------------------------------------------------ the module

def _module(dev, D=64, dt=F32, **kw):
    from memory_amd.memory_attention import MemoryCrossAttention
    torch.manual_seed(0)
    return MemoryCrossAttention(4 * D, 4, 2, memory_dim=96, wo_init_zero=False, **kw).to(dev).to(dt)


def _module_reference(m, h, mem, live, pos_q=None, pos_k=None):
    """The layer in float64 from its parameters."""
    W = {n: p.detach().double() for n, p in m.named_parameters()}
    h, mem = h.detach().double(), mem.detach().double()
    if mem.dim() == 2:
        mem = mem.expand(h.shape[0], *mem.shape)
    heads = lambda x, w, n: (x @ w.t()).view(*x.shape[:2], n, m.head_dim)
    q, k, v = heads(h, W["q_proj.weight"], 4), heads(mem, W["k_proj.weight"], 2), heads(mem, W["v_proj.weight"], 2)

    def treat(x, name, pos):
        if m.q_norm is not None:
            x = x * (x.square().mean(-1, keepdim=True) + getattr(m, name).eps).rsqrt() * W[name + ".weight"]
        R = m.rotary_dim
        if R:
            pos = torch.arange(x.shape[1], device=x.device) if pos is None else pos
            f = m.rotary_base ** (-torch.arange(0, R, 2, device=x.device, dtype=torch.float64) / R)
            a = pos.double()[..., None, None] * f
            u, w = x[..., :R // 2], x[..., R // 2:R]
            x = torch.cat([u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin(), x[..., R:]], -1)
        return x

    o = formula(treat(q, "q_norm", pos_q), treat(k, "k_norm", pos_k), v, live)
    return o.reshape(h.shape) @ W["o_proj.weight"].t()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(qk_norm=True), dict(rotary_dim=32), dict(qk_norm=True, rotary_dim=64),
                                dict(qk_norm=True, gradient_checkpointing=True)])
@pytest.mark.parametrize("D", [64, 128])
def test_module(gpu_device, D, kw):
    """float32 layer over ragged states against float64 (products of 256 or 512 terms and the attention: 1e-5 of the
    result's largest value covers (512 + 8) u for each of four chained products, 1.2e-4 would be their worst case)."""
    m = _module(gpu_device, D, **kw)
    g = gen(13)
    h = torch.randn(3, 21, 4 * D, generator=g).to(gpu_device).requires_grad_(True)
    mem = torch.randn(3, 50, 96, generator=g).to(gpu_device).requires_grad_(True)
    lens = torch.tensor([50, 7, 33], device=gpu_device)
    live = torch.arange(50, device=gpu_device)[None] < lens[:, None]
    pos = dict(query_positions=torch.arange(100, 121, device=gpu_device)) if kw.get("rotary_dim") else {}
    out, w = m(h, mem, memory_lengths=lens, **pos)
    ref = _module_reference(m, h, mem, live, pos.get("query_positions"))
    assert w is None and (out.double() - ref).abs().max() <= 1.2e-4 * ref.abs().max()
    by_mask, _ = m(h, mem, memory_mask=live, **pos)
    assert torch.equal(out, by_mask)
    params = [p for p in m.parameters()]
    grads = torch.autograd.grad(out.square().sum(), [h, mem, *params])
    assert all(torch.isfinite(x).all() and x.abs().max() > 0 for x in grads)
    assert (grads[1][1, 7:] == 0).all()


@pytest.mark.gpu
def test_module_shared_and_whole_tiles(gpu_device):
    """A 2-D memory of any length, and one of whole chapters with and without a mask that keeps every state."""
    m = _module(gpu_device)
    g = gen(14)
    h = torch.randn(2, 9, 256, generator=g).to(gpu_device)
    mem = torch.randn(45, 96, generator=g).to(gpu_device)
    every = torch.ones(2, 45, dtype=torch.bool, device=gpu_device)
    ref = _module_reference(m, h, mem, every)
    assert (m(h, mem)[0].double() - ref).abs().max() <= 1.2e-4 * ref.abs().max()
    mem = torch.randn(2, 128, 96, generator=g).to(gpu_device)
    every = torch.ones(2, 128, dtype=torch.bool, device=gpu_device)
    a, b = m(h, mem)[0], m(h, mem, memory_mask=every)[0]
    ref = _module_reference(m, h, mem, every)
    for x in (a, b):
        assert (x.double() - ref).abs().max() <= 1.2e-4 * ref.abs().max()


@pytest.mark.gpu
def test_sublayer(gpu_device):
    """MemorySublayer over masked states is residual + attention of the norm."""
    from memory_amd.memory_block import MemorySublayer
    torch.manual_seed(1)
    s = MemorySublayer(256, 4, 2, memory_dim=96, wo_init_zero=False, qk_norm=True, rotary_dim=64).to(gpu_device)
    h = torch.randn(2, 11, 256, generator=gen(15)).to(gpu_device)
    mem = torch.randn(2, 37, 96, generator=gen(16)).to(gpu_device)
    mask = (torch.rand(2, 37, generator=gen(17)) > 0.3).to(gpu_device)
    out = s(h, mem, memory_mask=mask, memory_positions=torch.arange(37, device=gpu_device) + 5)
    hd = h.double()
    normed = hd * (hd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    ref = hd + _module_reference(s.memory_attn, normed, mem, mask, None, torch.arange(37, device=gpu_device) + 5)
    assert (out.double() - ref).abs().max() <= 1.2e-4 * ref.abs().max()


@pytest.mark.gpu
def test_module_float16(gpu_device):
    m = _module(gpu_device, dt=torch.float16, qk_norm=True)
    h = torch.randn(2, 5, 256, generator=gen(18)).half().to(gpu_device)
    mem = torch.randn(2, 20, 96, generator=gen(19)).half().to(gpu_device)
    out, _ = m(h, mem, memory_lengths=torch.tensor([20, 4], device=gpu_device))
    assert out.dtype == torch.float16 and torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 4, 4, 2, 2, 64), (2, 200, 333, 4, 2, 64), (1, 30, 3000, 8, 2, 128), (3, 150, 150, 2, 1, 128)])
def test_backward_entry_without_some_gradients(gpu_device, shape, dt):
    """moc_cross_bwd gives dq alone, or dk and dv alone, to the bit of all three; it writes nothing else."""
    from memory_amd import _lib as L
    from memory_amd import ops
    B, Lq, N, H, HK, D = shape
    q, k, v, do = inputs(*shape, dt, gpu_device, seed=20)
    out, low, lse = ops._cross_forward(q, k, v, None, None, D ** -0.5, True)
    code = L.dtype_code(dt)
    nbytes = L.query("moc_cross_bwd_workspace", B, Lq, N, H, HK, D, code)

    def grads(want_q, want_kv):
        g = [torch.full_like(q, 7.0) if want_q else None, *(torch.full_like(k, 7.0) if want_kv else None for _ in range(2))]
        ws = torch.full((nbytes,), 0xff, device=gpu_device, dtype=torch.uint8)
        L.call("moc_cross_bwd", ops._pack_cross(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), do.data_ptr(), out.data_ptr(), ops.ptr0(low), *map(ops.ptr0, g), lse.data_ptr(),
            0, 0, *ops._strides3(q), *ops._strides3(k), *ops._strides3(v), *ops._strides3(do), B, Lq, N, H, HK, D, code, D ** -0.5),
            ws.data_ptr(), nbytes, L.stream_ptr(gpu_device))
        return g

    whole = grads(True, True)
    ref, bound = reference(q, k, v, None, do)
    for name, x, a, b in zip(("dq", "dk", "dv"), whole, ref[1:], bound[1:]):
        close(x, a, b, name)
    only_q, only_kv = grads(True, False), grads(False, True)
    assert torch.equal(only_q[0], whole[0]) and torch.equal(only_kv[1], whole[1]) and torch.equal(only_kv[2], whole[2])
    with pytest.raises(ValueError, match="null"):
        grads(False, False)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 200])
def test_largest_scale(gpu_device, L):
    """Logits of 0 under the largest scale: the mean of the values."""
    from memory_amd import ops
    q, k, v, _ = inputs(1, L, 5, 2, 1, 64, F32, gpu_device, seed=21)
    with torch.no_grad():
        o = ops.cross_attention(q, k * 0, v, softmax_scale=1.7e38)
    ref = v.double().mean(1, keepdim=True).expand_as(o)
    # (five probabilities and their sum, each exact but for the division, and five products and additions)
    assert ((o.double() - ref).abs() <= 16 * U * v.double().abs().mean(1, keepdim=True)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("power", [6, 12, 18, 24])
@pytest.mark.parametrize("B,L,N,copies,apart", [(1, 40, 60, 1, 1), (2, 300, 400, 1, 1), (1, 300, 400, 4, 1), (1, 7, 5000, 1, 1),
                                                (1, 1, 200, 2, 1), (1, 300, 400, 3, 130), (1, 7, 5000, 5, 999), (1, 1, 5000, 3, 7),
                                                (1, 130, 5000, 3, 1200)])
def test_one_key_takes_a_row(gpu_device, B, L, N, copies, apart, power, dt):
    """Logits of up to 2^power with one key, or equal copies of it ``apart`` keys from each other, far above the others (by
    more than 2^7, at 2^6 x 4): the weights are 1 / copies and 0, whatever the logits' own rounding.
      out  the copies' mean value (copies roundings of float32, then the result's), dv sum_i dO_i / copies (L + 64 of
           float32, then the weights' 2^-8 in bfloat16 calls of many rows and keys, and the result's),
      dq, dk of one copy: 0 up to what dP - delta, both sums of D terms, leaves of them: 2 (D + 8 + copies) u
           sum_d |dO_d v_d| (and 2^-16 of it in bfloat16: out's low piece) times scale |k|, |q|."""
    from memory_amd import ops
    D = 64
    g = gen(22)
    at = apart * torch.arange(copies)
    u = torch.sign(torch.randn(D, generator=g))
    q = (u * 2.0 ** ((power - 3) // 2)).expand(B, L, 1, D).contiguous()
    k = torch.randn(B, N, 1, 1, generator=g).clamp(-1, 1) * u * 2.0 ** ((power - 3) // 2) / 64
    k[:, at] = u * 2.0 ** (power - 3 - (power - 3) // 2) * (1 if power > 6 else 4)
    v, do = torch.randn(B, N, 1, D, generator=g), torch.randn(B, L, 1, D, generator=g)
    q, k, v, do = (x.to(dt).to(gpu_device) for x in (q, k, v, do))
    s = (q[0, :1, 0].double() @ k[0, :, 0].double().t().contiguous())[0] / 8
    rest = torch.ones(N, dtype=torch.bool)
    rest[at] = False
    assert (s[at] == s.max()).all() and s.max() - s[rest].max() > 128
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = ops.cross_attention(q, k, v)
    with torch.no_grad():
        served = ops.cross_attention(q, k, v)
    dq, dk, dv = torch.autograd.grad(o, [q, k, v], do)
    t = 2.0 ** -24 if dt == F32 else 2.0 ** -8
    r = 2.0 ** -8 if dt == BF and min(N, L) > 128 else 0.0 if dt == F32 else 2.0 ** -16
    vd, dod = v.detach().double(), do.double()
    mean, mag = vd[:, at].mean(1, keepdim=True), vd[:, at].abs().mean(1, keepdim=True)
    for name, x in (("out", o.detach()), ("served", served)):
        close(x, mean.expand_as(o), (t * mean.abs() + (2 * copies + 64) * U * mag).expand_as(o), name)
    want, bound = torch.zeros_like(vd), torch.zeros_like(vd)
    want[:, at] = dod.sum(1, keepdim=True) / copies
    bound[:, at] = (t * dod.sum(1, keepdim=True).abs() + (r + (L + 64) * U) * dod.abs().sum(1, keepdim=True)) / copies
    close(dv, want, bound, "dv")
    if copies == 1:
        noise = (2 * (D + 8 + copies) * U + (2.0 ** -16 if dt == BF else 0.0))
        left = noise * (dod.abs() * vd[:, :1].abs()).sum(-1, keepdim=True)          # (B, L, 1, 1)
        close(dq, torch.zeros_like(dod), left / 8 * k.detach().double()[:, :1].abs(), "dq")
        close(dk[:, :1], torch.zeros_like(vd[:, :1]), (left / 8 * q.detach().double().abs()).sum(1, keepdim=True), "dk")
        assert (dk[:, 1:] == 0).all()
        if dt == F32 or min(N, L) <= 128:
            assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", [(2, 7, 1, 8, 2, 64), (1, 300, 1, 4, 1, 128), (3, 150, 1, 2, 2, 64), (1, 1, 1, 1, 1, 128)])
def test_single_key(gpu_device, shape, dt):
    """Over one key the result is its value to the bit, and dq and dk are exactly 0 (dP and delta are one sum, formed
    alike), not its rounding."""
    q, k, v, do = inputs(*shape, dt, gpu_device, seed=23, train=True)
    o, dq, dk, dv = check(q, k, v, do)
    G = shape[3] // shape[4]
    assert torch.equal(o, v.detach().repeat_interleave(G, 2).expand_as(o))
    assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.gpu
def test_sublayer_attention_alone(gpu_device):
    """What MemorySublayer adds to the residual, against the attention's own largest value: four chained products of at
    most 256 terms and the attention, (512 + 8) u each at worst (1.2e-4), and the rounding of the sum."""
    from memory_amd.memory_block import MemorySublayer
    torch.manual_seed(4)
    s = MemorySublayer(256, 4, 2, memory_dim=96, wo_init_zero=False, qk_norm=True, rotary_dim=64).to(gpu_device)
    h = torch.randn(2, 11, 256, generator=gen(24)).to(gpu_device)
    mem = torch.randn(2, 37, 96, generator=gen(25)).to(gpu_device)
    lens = torch.tensor([37, 5], device=gpu_device)
    with torch.no_grad():
        out = s(h, mem, memory_lengths=lens).double()
    hd = h.double()
    normed = hd * (hd.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    live = torch.arange(37, device=gpu_device)[None] < lens[:, None]
    ref = _module_reference(s.memory_attn, normed, mem, live)
    assert ((out - hd - ref).abs() <= 1.2e-4 * ref.abs().max() + U * out.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L,N", [(1, 40), (1, 5000), (40, 60), (7, 5000), (300, 400), (200, 5000)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_go_through(gpu_device, L, N, bad, dt):
    """NaN or infinity in a key that counts, alone in its split too, makes NaN of every row of its kv head and of no
    other; one in a query, of its row; a NaN in a value, of its column."""
    from memory_amd import ops
    q, k, v, do = inputs(2, L, N, 4, 2, 64, dt, gpu_device, seed=26)
    q = q.abs()
    k[0, N - 1, 0] = bad          # (every term of its logits is NaN or +inf)
    q[1, L // 2, 3, 5] = float("nan")
    v[1, N // 2, 0, 9] = float("nan")
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    with torch.no_grad():
        served = ops.cross_attention(q, k, v)
    trained = ops.cross_attention(q, k, v)
    want = torch.zeros(2, L, 4, 64, dtype=torch.bool, device=gpu_device)
    want[0, :, :2] = True
    want[1, L // 2, 3] = True
    want[1, :, :2, 9] = True
    for name, o in (("served", served), ("trained", trained.detach())):
        assert torch.equal(torch.isnan(o), want), name
    dq, dk, dv = torch.autograd.grad(trained, [q, k, v], do)
    assert torch.isnan(dq[0, :, :2]).all() and torch.isfinite(dq[0, :, 2:]).all()
    assert torch.isnan(dq[1, L // 2, 3]).all() and torch.isfinite(dq[1, :, 2]).all()
    assert torch.isfinite(dk[0, :, 1]).all() and torch.isfinite(dv[0, :, 1]).all()
    assert torch.isnan(dv[0, :, 0]).all() and torch.isnan(dv[1, :, 1]).all()
