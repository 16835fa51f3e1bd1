"""The sublayer's operators in one run, as they are used together: expert-style routing, the memory attention, the norms
around it with gate and residual scale; trained (every gradient against float64), and served from an 8-bit cache
token by token and for a prompt.  Gates of tests/helpers.py: float32 1e-4, bfloat16 2e-2."""

import pytest
import torch

import oracle as O
from helpers import assert_parity, gen
from test_gpu_router_select import reference

pytestmark = pytest.mark.gpu
BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
OPTIONS = dict(score="sigmoid", num_groups=4, top_groups=2, balance_bias=True)


def norm64(x, w, b, eps, rms):
    if rms:
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    return torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b, eps)


def build(dev, dtype, rms, d, H, HK, C, k, gate, seed):
    from memory_amd.memory_block import MemorySublayer, RMSNorm
    from memory_amd.router import ChapterRouter
    g0 = gen(seed)
    r = lambda *s, std=1.0, mean=0.0: torch.randn(*s, generator=g0) * std + mean
    router = ChapterRouter(d, C, k, **OPTIONS)
    sub = MemorySublayer(d, H, HK, use_rms_norm=rms, norm_eps=1e-5, wo_init_zero=False, post_norm=True, gate=gate,
                         residual_scale=0.8)
    nxt = RMSNorm(d, 1e-6) if rms else torch.nn.LayerNorm(d, eps=1e-6)
    with torch.no_grad():
        router.router.weight.copy_(r(C, d, std=0.1))
        router.balance_bias.copy_(r(C, std=0.05))
        for ln in (sub.memory_layernorm, sub.post_layernorm, nxt):
            ln.weight.copy_(r(d, std=0.2, mean=1.0))
            if not rms:
                ln.bias.copy_(r(d, std=0.1))
        sub.gate.copy_(r(*sub.gate.shape, std=0.3, mean=0.6))
        for lin in (sub.memory_attn.q_proj, sub.memory_attn.k_proj, sub.memory_attn.v_proj, sub.memory_attn.o_proj):
            lin.weight.copy_(r(*lin.weight.shape, std=d ** -0.5).to(dtype).float())
    for m in (router, sub, nxt):
        m.to(dev)
    for lin in (sub.memory_attn.q_proj, sub.memory_attn.k_proj, sub.memory_attn.v_proj, sub.memory_attn.o_proj):
        lin.to(dtype)
    return router, sub, nxt, g0


def weights64(router, sub, nxt):
    a = sub.memory_attn
    names = dict(Wr=router.router.weight, br=router.router.bias, n1=sub.memory_layernorm.weight, p1=sub.post_layernorm.weight,
                 x1=nxt.weight, gate=sub.gate, Wq=a.q_proj.weight, Wk=a.k_proj.weight, Wv=a.v_proj.weight, Wo=a.o_proj.weight)
    if not sub.use_rms_norm:
        names.update(n1b=sub.memory_layernorm.bias, p1b=sub.post_layernorm.bias, x1b=nxt.bias)
    return names, {k: p.detach().cpu().double().requires_grad_(True) for k, p in names.items()}


@pytest.mark.parametrize("dtype,rms,gate,HK", [(F32, True, "channel", 4), (F32, False, "scalar", 2), (BF, True, "channel", 2),
                                               (BF, False, "scalar", 4)])
def test_training_step(gpu_device, dtype, rms, gate, HK):
    from memory_amd.model import prepend_shared_chapters32
    dev, B, L, d, H, C, T, k, S = gpu_device, 3, 70, 256, 4, 17, 64, 3, 1
    router, sub, nxt, g0 = build(dev, dtype, rms, d, H, HK, C, k, gate, 31 + rms)
    h = torch.randn(B, L, d, generator=g0).to(dtype)
    bank = (torch.randn(C * T, d, generator=g0) * 0.5).to(dtype)
    d1, d2 = torch.randn(B, L, d, generator=g0), torch.randn(B, L, d, generator=g0)
    hg, bg = h.to(dev).requires_grad_(True), bank.to(dev).requires_grad_(True)
    idx, w, losses = router.route_ids32(hg, exclude_prefix_chapters=S)
    ci, om = prepend_shared_chapters32(idx, w, num_chapters=C, num_shared_chapters=S, routed_scaling_factor=2.5)
    state = {"bank": bg, "chapter_indices": ci, "chapter_weights": om, "num_chapters": C, "tokens_per_chapter": T}
    out, nrm = sub(hg, routed_memory_state=state, next_norm=nxt)
    assert out.dtype == nrm.dtype == dtype and losses
    ((out.float() * d1.to(dev)).sum() + (nrm.float() * d2.to(dev)).sum()).backward()

    names, w64 = weights64(router, sub, nxt)
    h64, b64 = h.double().requires_grad_(True), bank.double().requires_grad_(True)
    g = lambda n: w64.get(n)
    logits = h64.mean(1) @ w64["Wr"].t() + w64["br"]
    ridx, _, _ = reference(logits, k, S, "sigmoid", router.balance_bias.cpu(), 4, 2)
    assert torch.equal(idx.cpu(), ridx)
    s = torch.sigmoid(logits).gather(1, ridx.long())
    rw = s / s.sum(1, keepdim=True)
    rci, rom = O.prepend_shared_chapters(ridx.long(), rw, num_chapters=C, num_shared_chapters=S,
                                         routed_scaling_factor=2.5)
    rom.retain_grad()
    mem = O.weight_memory(O.gather_chapters(b64, rci, T)[0], rom, T)
    x = norm64(h64, w64["n1"], g("n1b"), 1e-5, rms)
    att = O.attention((x @ w64["Wq"].t()).view(B, L, H, 64), (mem @ w64["Wk"].t()).view(B, -1, HK, 64).repeat_interleave(H // HK, 2),
                      (mem @ w64["Wv"].t()).view(B, -1, HK, 64).repeat_interleave(H // HK, 2)).reshape(B, L, -1)
    u = norm64(att @ w64["Wo"].t(), w64["p1"], g("p1b"), 1e-5, rms)
    ref = 0.8 * h64 + w64["gate"] * u
    refn = norm64(ref, w64["x1"], g("x1b"), 1e-6, rms)
    ((ref * d1.double()).sum() + (refn * d2.double()).sum()).backward()
    assert_parity(out.float(), ref.detach(), dtype, "hidden")
    assert_parity(nrm.float(), refn.detach(), dtype, "next norm")
    assert_parity(hg.grad.float(), h64.grad, dtype, "dh")
    assert_parity(bg.grad.float(), b64.grad, dtype, "dbank")
    for n, p in names.items():
        if dtype == F32 or n not in ("Wr", "br"):
            assert_parity(p.grad.float(), w64[n].grad, dtype, "d" + n)
    if dtype == BF:
        # The router's gradient is a difference of the attention's gradients of omega, which renormalising the weights
        # takes out the common part of: with omega's gradient within the bfloat16 gate (2e-2 of its maximum), a logit's
        # is within 2e-2 max|d omega| sum_j |d omega_j / d logit|, the bias' within the rows' sum of that, the weight's
        # within that sum times the pooled states.
        bound = torch.zeros(B, C, dtype=torch.float64)
        for b in range(B):
            def omega_of(z):
                sel = torch.sigmoid(z)[ridx[b].long()]
                om = torch.cat([torch.ones(S, dtype=torch.float64), 2.5 * sel / sel.sum()])
                return om / om.sum()
            jac = torch.autograd.functional.jacobian(omega_of, logits[b].detach())
            bound[b] = 2e-2 * rom.grad.abs().max() * jac.abs().sum(0)
        pooled = h64.detach().mean(1)
        assert torch.allclose(omega_of(logits[b].detach()), rom[b].detach())
        err_b = (names["br"].grad.cpu().double() - w64["br"].grad).abs()
        err_w = (names["Wr"].grad.cpu().double() - w64["Wr"].grad).abs()
        print(f"router gradient: {(err_b / (bound.sum(0) + 1e-12)).max():.3f}, {(err_w / (bound.t() @ pooled.abs() + 1e-12)).max():.3f}")
        assert (err_b <= bound.sum(0) + 1e-12).all() and (err_w <= bound.t() @ pooled.abs() + 1e-12).all()
    # the balance step
    before = router.balance_bias.clone()
    counts = router.update_balance(idx, 0.01, S)
    assert counts.sum() == idx.numel() and counts[:S].sum() == 0
    moved = torch.sign(counts[S:].double().mean() - counts[S:].double()) * 0.01
    assert torch.equal(router.balance_bias[S:], before[S:] + moved.float()) and torch.equal(router.balance_bias[:S], before[:S])


def test_layers_take_the_options(gpu_device):
    """RoutedMemoryLayer, TokenRoutedMemoryLayer, MemoryStack and DecodeRouter with an expert-style router select as the
    operator does; a plain router keeps the fused path; state dicts carry the bias only where there is one."""
    from memory_amd import ops
    from memory_amd.checkpoint import MemoryStack
    from memory_amd.decode import DecodeRouter
    from memory_amd.model import RoutedMemoryLayer, TokenRoutedMemoryLayer
    from memory_amd.router import ChapterRouter
    dev, d, H, C, k = gpu_device, 256, 4, 33, 4
    h = torch.randn(2, 24, d, generator=gen(1)).to(dev, BF)
    bank = (torch.randn(C * 64, d, generator=gen(2)) * 0.5).to(dev, BF)
    for cls in (RoutedMemoryLayer, TokenRoutedMemoryLayer):
        plain, lay = cls(d, H, C, 64, k).to(dev), cls(d, H, C, 64, k, router_options=OPTIONS).to(dev)
        assert plain.router.plain_selection and not lay.router.plain_selection
        assert set(lay.state_dict()) - set(plain.state_dict()) == {"router.balance_bias"}
        for m in (plain, lay):
            m.memory_attn.to(BF)
        with torch.no_grad():
            lay.router.balance_bias.copy_(torch.randn(C, generator=gen(3)) * 0.1)
        out, losses = lay(h, bank)
        assert out.shape == h.shape and losses
        out.float().square().sum().backward() if out.requires_grad else None
        pooled = h.float().mean(1) if cls is RoutedMemoryLayer else h.reshape(-1, d)
        if cls is RoutedMemoryLayer:
            idx, w, _ = lay.router(h, exclude_prefix_chapters=1)
            logits = ops.router_linear(ops.router_pool(h), lay.router.router.weight, lay.router.router.bias)
        else:
            idx, w, _ = lay.router.route_token_level(h, exclude_prefix_chapters=1)
            logits = ops.router_token_logits(h, lay.router.router.weight, lay.router.router.bias)
        ridx, rw, _ = reference(logits, k, 1, "sigmoid", lay.router.balance_bias.cpu(), 4, 2)
        assert torch.equal(idx.reshape(-1, k).cpu().int(), ridx)
        assert (w.reshape(-1, k).cpu().double() - rw).abs().max() <= 2.0 ** -16
        assert pooled is not None
    r = ChapterRouter(d, C, k, **OPTIONS).to(dev)
    dr = DecodeRouter(r, num_chapters=C, strategy="rolling", window_size=8)
    dr.prefill(h)
    route = dr.step(h[:, -1:])
    ridx, rw, _ = reference(dr.last_logits, k, 1, "sigmoid", r.balance_bias.cpu(), 4, 2)
    assert torch.equal(route.idx[:, 1:].cpu(), ridx) and not route.idx[:, 0].any()
    om = torch.cat([torch.ones(2, 1), 2.5 * rw.float()], 1)
    assert (route.omega.cpu() - om / om.sum(1, keepdim=True)).abs().max() <= 2.0 ** -16
    mem = dict(use_chapters=True, num_chapters=C, num_memory_tokens=C * 64, top_k_chapters=k, num_shared_chapters=1,
               router_options=OPTIONS)
    stack = MemoryStack(hidden_dim=d, num_layers=1, num_heads=H, num_kv_heads=None, memory=mem)
    sd = {n: v for n, v in stack.state_dict().items() if not n.endswith("balance_bias")}
    stack.load_reference_state_dict(sd)
    stack.to(dev)
    out, _ = stack(0, h.float(), h.float())
    assert out.shape == h.shape


@pytest.mark.parametrize("HK", [4, 1])
def test_serving_from_an_8_bit_cache(gpu_device, HK):
    """A prompt and then tokens with routing decided by the expert-style router at each of them: q projection,
    attention over the 8-bit cache, o projection, post-norm, gate, residual and the next norm, against float64 on the values
    the cache stands for; and the same step captured and replayed."""
    from memory_amd.decode import DecodeRouter, DecodeStepGraph, MemoryDecodeCache, memory_decode_step
    dev, B, d, H, C, k, S = gpu_device, 5, 256, 4, 33, 6, 1
    router, sub, nxt, g0 = build(dev, BF, True, d, H, HK, C, k, "channel", 7)
    for p in (*router.parameters(), *sub.parameters(), *nxt.parameters()):
        p.requires_grad_(False)
    bank = (torch.randn(C * 64, d, generator=g0) * 0.5).to(dev, BF)
    attn = sub.memory_attn
    cache = MemoryDecodeCache(bank, attn.k_proj.weight, attn.v_proj.weight, num_chapters=C, tokens_per_chapter=64,
                              num_kv_heads=HK, dtype=FP8)
    K, V = (t.cpu().double() for t in cache.dequantized())
    dr = DecodeRouter(router, num_chapters=C, num_shared_chapters=S, strategy="rolling", window_size=16)
    _, w64 = weights64(router, sub, nxt)
    w64 = {n: t.detach() for n, t in w64.items()}

    def step(x, routing):
        normed = sub.memory_layernorm(x)
        return sub.join(memory_decode_step(attn, normed, cache, routing), x, nxt)

    def want(x, routing):
        x = x.cpu().double()
        Lx, idx, om = x.shape[1], routing.idx.cpu().long(), routing.omega.cpu().double()
        q = (norm64(x, w64["n1"], None, 1e-5, True) @ w64["Wq"].t()).view(B, Lx, H, 64)
        kk = (K[idx] * om[..., None, None, None]).transpose(2, 3).reshape(B, -1, HK, 64).repeat_interleave(H // HK, 2)
        vv = (V[idx] * om[..., None, None, None]).transpose(2, 3).reshape(B, -1, HK, 64).repeat_interleave(H // HK, 2)
        att = O.attention(q, kk, vv).reshape(B, Lx, -1)
        hid = 0.8 * x + w64["gate"] * norm64(att @ w64["Wo"].t(), w64["p1"], None, 1e-5, True)
        return hid, norm64(hid, w64["x1"], None, 1e-6, True)

    prompt = torch.randn(B, 19, d, generator=g0).to(dev, BF)
    routing = dr.prefill(prompt)
    for x in [prompt] + [torch.randn(B, 1, d, generator=g0).to(dev, BF) for _ in range(3)]:
        if x.shape[1] == 1:
            routing = dr.step(x)
        got, ref = step(x, routing), want(x, routing)
        for name, a, b in zip(("hidden", "next norm"), got, ref):
            assert a.shape == x.shape and a.dtype == BF
            assert_parity(a.float(), b, BF, name)
    graph = DecodeStepGraph([(attn, cache, routing)], [x])
    for rep in range(3):
        y = torch.randn(B, 1, d, generator=gen(rep)).to(dev, BF)
        a = graph.run([y])[0].clone()
        torch.cuda.synchronize()
        assert torch.equal(a, memory_decode_step(attn, y, cache, routing))


def test_sublayer_forms(gpu_device):
    """A gate of the caller's own (per row, per element), rows normed by the previous sublayer, and the plain sublayer
    unchanged by the options' defaults."""
    from memory_amd import ops
    from memory_amd.memory_block import MemorySublayer, RMSNorm
    dev, B, L, d, H = gpu_device, 2, 9, 256, 4
    torch.manual_seed(0)
    h = torch.randn(B, L, d).to(dev)
    mem = torch.randn(B, 128, d).to(dev)
    plain = MemorySublayer(d, H, wo_init_zero=False).to(dev)
    assert set(plain.state_dict()) == {"memory_layernorm.weight"} | {f"memory_attn.{n}_proj.weight" for n in "qkvo"}
    base = plain(h, mem)
    nxt = RMSNorm(d).to(dev)
    out, n = plain(h, mem, next_norm=nxt)
    assert (out - base).abs().max() <= 1e-5 * base.abs().max()
    assert (n - ops.row_norm(out, nxt.weight, None, nxt.eps)).abs().max() <= 1e-5
    out2 = plain(h, mem, normed=plain.memory_layernorm(h))
    assert (out2 - base).abs().max() <= 1e-4 * base.abs().max()
    for gate in (torch.rand(B, L, 1, device=dev), torch.rand(B, L, d, device=dev)):
        got = plain(h, mem, gate=gate)
        assert (got - (h + gate * (base - h))).abs().max() <= 1e-5 * base.abs().max()
    with pytest.raises(ValueError):
        MemorySublayer(d, H, gate="token")
    with pytest.raises(ValueError):
        plain(h, mem, next_norm=torch.nn.Identity())
    half = MemorySublayer(d, H, wo_init_zero=False, post_norm=True, gate="scalar").to(dev).half()
    o16, n16 = half(h.half(), mem.half(), next_norm=nxt)
    assert o16.dtype == n16.dtype == torch.float16


def test_balance_from_the_last_training_step(gpu_device):
    """update_balance without ids counts the last selection made in training mode, and no other."""
    from memory_amd.model import RoutedMemoryLayer, TokenRoutedMemoryLayer
    dev, d, H, C, k = gpu_device, 128, 2, 17, 4
    bank = (torch.randn(C * 64, d, generator=gen(2)) * 0.5).to(dev)
    for cls, rows in ((RoutedMemoryLayer, 3), (TokenRoutedMemoryLayer, 3 * 20)):
        lay = cls(d, H, C, 64, k, router_options=dict(score="sigmoid", balance_bias=True)).to(dev)
        router = lay.router
        with pytest.raises(ValueError):
            router.update_balance()
        h = torch.randn(3, 20, d, generator=gen(4)).to(dev)
        out, _ = lay(h, bank)
        out.sum().backward()
        seen = router.selected.clone()
        assert seen.shape == (rows, k)
        lay.eval()
        lay(torch.randn(5, 20, d, generator=gen(5)).to(dev), bank)
        assert torch.equal(router.selected, seen)
        counts = router.update_balance(rate=0.5, exclude_prefix_chapters=1)
        want = torch.bincount(seen.reshape(-1).cpu().long(), minlength=C)
        assert torch.equal(counts.cpu().long(), want)
        moved = 0.5 * torch.sign(want[1:].double().mean() - want[1:].double())
        assert torch.equal(router.balance_bias[1:].cpu().double(), moved) and router.balance_bias[0] == 0
        plain = cls(d, H, C, 64, k).to(dev)
        plain(h, bank)
        assert plain.router.selected is None
