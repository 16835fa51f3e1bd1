"""The decode cache in 8 bits (e4m3 tiles with one scale per chapter and kv head): its quantisation bit by bit, and
the attention over it against float64.

Tolerances, derived: the products run on exact operands (bfloat16 queries, e4m3 values widened exactly) with float32
sums; probabilities are rounded to bfloat16 (2^-8 each), part rows of a chapter once more, the result once, and row
sums may carry the probabilities' rounding: 2^-8 |o| + 3 2^-8 sum_j p_j |v_j|.  A logit's float32 sum of 64 products is off
by at most 64 2^-24 sum |q k|, which moves a probability by as much: 2^-17 times the largest logit's terms."""

import math

import pytest
import torch

from helpers import gen

BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
H8 = 2.0 ** -8


def make_tiles(C, HK, seed, spread=0.5):
    g0 = gen(seed)
    x = torch.randn(C, HK, 64, 64, generator=g0) * torch.exp(spread * torch.randn(C, HK, 1, 1, generator=g0))
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)).double() / 448))).float()
    return (x / s[:, :, None, None]).to(FP8), s


def reference(q, k8, ks, v8, vs, idx, omega):
    """(o, bound) float64 of q (B, L, H, 64); slots whose id is out of range are left out."""
    B, Lq, H, D = q.shape
    C, HK = ks.shape
    out, bound = torch.zeros(B, Lq, H, D, dtype=torch.float64), torch.zeros(B, Lq, H, D, dtype=torch.float64)
    for b in range(B):
        sl = [s for s in range(idx.shape[1]) if 0 <= int(idx[b, s]) < C]
        if not sl:
            continue
        ids = idx[b, sl].long()
        om = omega[b, sl].double()
        k = k8[ids].to(F32).double() * ks[ids].double()[:, :, None, None] * om[:, None, None, None]
        v = v8[ids].to(F32).double() * vs[ids].double()[:, :, None, None] * om[:, None, None, None]
        for h in range(H):
            kk, vv = k[:, h // (H // HK)].reshape(-1, D), v[:, h // (H // HK)].reshape(-1, D)
            qd = q[b, :, h].double()
            p = torch.softmax(qd @ kk.t() / 8, dim=1)
            out[b, :, h] = p @ vv
            mag = p @ vv.abs()
            logit = (qd.abs() @ kk.abs().t() / 8).amax(1, keepdim=True)
            bound[b, :, h] = H8 * out[b, :, h].abs() + (3 * H8 + 2.0 ** -16 * logit) * mag
    return out, bound


def make(B, L, H, HK, C, NS, seed, distinct=True):
    g0 = gen(seed)
    k8, ks = make_tiles(C, HK, seed + 1)
    v8, vs = make_tiles(C, HK, seed + 2)
    q = torch.randn(B, L, H, 64, generator=g0).to(BF)
    if distinct and NS <= C:
        idx = torch.stack([torch.randperm(C, generator=g0)[:NS] for _ in range(B)]).int()
    else:
        idx = torch.randint(0, C, (B, NS), generator=g0).int()
    omega = torch.rand(B, NS, generator=g0) * 1.5
    return q, k8, ks, v8, vs, idx, omega


def attend(dev, q, k8, ks, v8, vs, idx, omega, sync=True):
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    C, HK = ks.shape
    cache = MemoryDecodeCache.from_tiles(k8.to(dev), v8.to(dev), num_chapters=C, tokens_per_chapter=64, num_kv_heads=HK,
                                         k_scale=ks.to(dev), v_scale=vs.to(dev))
    routing = DecodeRouting(idx.to(dev), omega.to(dev), C, sync=sync)
    qd = q.to(dev)
    out = decode_attention(qd[:, 0] if q.shape[1] == 1 else qd, cache, routing)
    assert out.dtype == BF
    return out.view(q.shape)


def check(got, q, k8, ks, v8, vs, idx, omega):
    want, bound = reference(q, k8, ks, v8, vs, idx, omega)
    err = (got.cpu().double() - want).abs()
    worst = (err / (bound + 1e-30)).max().item() if err.numel() else 0
    print(f"q {tuple(q.shape)} C={ks.shape[0]} HK={ks.shape[1]} NS={idx.shape[1]}: worst {worst:.3f} of the bound", flush=True)
    assert (err <= bound + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF])
def test_pack(gpu_device, dtype):
    """Scales and bytes equal the definition's, on ordinary tiles and on zeros, infinities, NaN, magnitudes at a
    scale's edge, subnormal and huge ones."""
    from memory_amd.decode import MemoryDecodeCache, _v8_natural
    g0 = gen(1)
    C, HK = 12, 3
    k = torch.randn(C, HK, 64, 64, generator=g0) * torch.exp(3 * torch.randn(C, HK, 1, 1, generator=g0))
    v = torch.randn(C, HK, 64, 64, generator=g0)
    k[0, 0] = 0
    k[0, 1].clamp_(-1, 1)[3, 4] = 448.0
    k[0, 2].clamp_(-1, 1)[3, 4] = -450.0
    k[1, 0].clamp_(-1, 1)[63, 63] = 256.0
    k[1, 1, 5, 6] = float("inf")
    k[1, 1, 7, 8] = float("-inf")
    k[1, 2, 0, 0] = float("nan")
    k[2, 0] = float("nan")
    k[2, 1] *= 1e-30
    k[2, 2] = k[2, 2].clamp(-3, 3) * 1e37
    k[3, 0] = torch.randn(64, 64, generator=g0) * 1e-39 if dtype == F32 else 0
    k[3, 1] = float("inf")
    k, v = k.to(dtype), v.to(dtype)
    cache = MemoryDecodeCache.from_tiles(k.to(gpu_device), v.to(gpu_device), num_chapters=C, tokens_per_chapter=64,
                                         num_kv_heads=HK).quantized()
    for x, tiles, scale in ((k, cache.k_tiles, cache.k_scale), (v, _v8_natural(cache.v_tiles), cache.v_scale)):
        x = x.double()
        fin = torch.where(x.isfinite(), x.abs(), 0.0).amax((2, 3))
        e = torch.where(fin > 0, torch.ceil(torch.log2(fin / 448)), 0.0)
        # log2 of 448 2^e itself may round either way: decide by the definition
        e = torch.where((fin > 0) & (fin > 448 * torch.exp2(e)), e + 1, e)
        e = torch.where((fin > 0) & (fin <= 448 * torch.exp2(e - 1)), e - 1, e).clamp(-120, 120)
        assert torch.equal(scale.cpu().double(), torch.exp2(e))
        y = (x / torch.exp2(e)[:, :, None, None]).clamp(-448, 448).float().to(FP8)
        got = tiles.cpu()
        nan = x.isnan()
        assert got.float()[nan].isnan().all()
        assert torch.equal(got.float()[~nan], y.float()[~nan])
    kd, vd = cache.dequantized()
    assert kd.shape == (C, HK, 64, 64) and torch.equal(vd.cpu(), (y.float() * scale.cpu()[:, :, None, None]))
    assert cache.nbytes == 2 * C * HK * 4096 + 8 * C * HK and cache.quantized() is cache


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,HK,C,NS", [(1, 1, 1, 1, 1, 1), (1, 1, 12, 12, 65, 65), (3, 1, 8, 1, 20, 5), (5, 1, 16, 4, 40, 33),
                                           (64, 1, 4, 2, 33, 9), (2, 1, 32, 2, 10, 70), (40, 1, 12, 4, 8, 5), (300, 1, 2, 1, 9, 3),
                                           (2, 2, 4, 4, 20, 7), (3, 3, 8, 2, 20, 65), (2, 16, 2, 2, 9, 4), (1, 17, 2, 2, 9, 4),
                                           (2, 5, 16, 4, 30, 12), (1, 33, 16, 1, 30, 65), (2, 129, 4, 2, 12, 9), (1, 509, 4, 4, 70, 65),
                                           (3, 300, 8, 8, 9, 1), (1, 2, 64, 1, 5, 3), (1, 1000, 3, 3, 7, 2)])
def test_attention(gpu_device, B, L, H, HK, C, NS):
    case = make(B, L, H, HK, C, NS, B + L + H + C)
    check(attend(gpu_device, *case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 4, 40])
def test_slots_weights_and_scales(gpu_device, L):
    """Skipped slots (ids out of range), rows without any slot, a chapter chosen twice, weights of 0, scales that are
    no powers of two, 0, or far from 1."""
    q, k8, ks, v8, vs, idx, omega = make(6, L, 4, 2, 12, 8, 5, distinct=False)
    idx[0, 2], idx[0, 5], idx[1, 0] = -1, 12, 2 ** 31 - 1
    idx[2] = -7
    idx[3] = 4
    omega[4, :3] = 0
    omega[5] = 0
    ks = ks * (0.5 + torch.rand(12, 2, generator=gen(3)))
    vs = vs * (0.5 + torch.rand(12, 2, generator=gen(4)))
    ks[3], vs[5], ks[7], vs[7] = 0.0, 0.0, 1e-30, 1e-30
    vs[8], vs[9] = 1e30, 1e-35
    case = (q, k8, ks, v8, vs, idx, omega)
    for sync in (True, False):
        got = attend(gpu_device, *case, sync=sync)
        check(got, *case)
        assert not got[2].any() and not got[5].any()
    none = (q, k8, ks, v8, vs, torch.full_like(idx, -1), omega)
    assert not attend(gpu_device, *none).any()


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 24])
def test_value_factors_far_apart_and_long_tails(gpu_device, L):
    """Value factors over twenty powers of two in one sequence, the largest on a chapter that hardly counts, and
    probabilities of 2^-13 of the largest whose sum is an eighth of it: none may be rounded away."""
    C = 24
    q, k8, ks, v8, vs, idx, omega = make(3, L, 4, 2, C, C, 12)
    k, q = torch.zeros(C, 2, 64, 64), q.abs().clamp(0.5, 1)
    q[..., 0] = 8
    k[:, :, 1:, 0] = -9.0            # logit -9 beside one key's 0 in chapter 5: e^-9 = 2^-13
    k[:, :, 0, 0] = -9.0
    k[5, :, 7, 0] = 0.0
    k[0] = 0
    k[0, :, :, 0] = -30.0
    omega = torch.ones_like(omega)
    vs = torch.full((C, 2), 2.0 ** -11)
    vs[0], vs[11], vs[17] = 1.0, 2.0 ** -5, 2.0 ** -20
    case = (q, k.to(FP8), torch.ones(C, 2), v8.float().abs().to(FP8), vs, idx, omega)
    check(attend(gpu_device, *case), *case)
    for order in (idx.sort(1).values, idx.sort(1, descending=True).values):
        case = (*case[:5], order, omega)
        check(attend(gpu_device, *case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 24])
def test_large_logits_and_nan(gpu_device, L):
    """Logits of several hundred (one key takes all), and a NaN that stays in the sequences and heads that read it."""
    case = list(make(3, L, 4, 2, 10, 4, 8))
    case[2] = case[2] * 60
    check(attend(gpu_device, *case), *case)
    clean = attend(gpu_device, *case)
    k8 = case[1].view(torch.uint8).clone()
    hit = int(case[5][1, 2])
    k8[hit, 1, 3, 3] = 0x7f
    case[1] = k8.view(FP8)
    got = attend(gpu_device, *case)
    for b in range(3):
        reads = hit in case[5][b].tolist()
        assert torch.equal(got[b, :, :2], clean[b, :, :2])
        assert got[b, :, 2:].isnan().all() if reads else torch.equal(got[b], clean[b])


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 6, 70])
def test_query_layouts_and_types(gpu_device, L):
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    q, k8, ks, v8, vs, idx, omega = make(2, L, 4, 2, 9, 5, 3)
    want = attend(gpu_device, q, k8, ks, v8, vs, idx, omega)
    cache = MemoryDecodeCache.from_tiles(k8.to(gpu_device), v8.to(gpu_device), num_chapters=9, tokens_per_chapter=64,
                                         num_kv_heads=2, k_scale=ks.to(gpu_device), v_scale=vs.to(gpu_device))
    routing = DecodeRouting(idx.to(gpu_device), omega.to(gpu_device), 9)
    qd = q.to(gpu_device)
    views = [qd.float(), qd.transpose(1, 2).contiguous().transpose(1, 2), qd.half().float().half()]
    off = torch.zeros(qd.numel() + 3, device=gpu_device, dtype=BF)[3:].view(q.shape).copy_(qd)
    for v in views[:2] + [off]:
        got = decode_attention(v[:, 0] if L == 1 else v, cache, routing).view(q.shape)
        assert torch.equal(got, want)
    assert decode_attention(qd[:, :0], cache, routing).shape == (2, 0, 4, 64)


@pytest.mark.gpu
def test_tiles_past_four_gib(gpu_device):
    """A cache whose last tiles lie past 2^32 bytes."""
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    C, HK = 16384, 66
    q, k8, ks, v8, vs, idx, omega = make(2, 1, HK, HK, 4, 4, 9)
    tiles = torch.zeros(C, HK, 64, 64, device=gpu_device, dtype=torch.uint8)
    scale = torch.ones(C, HK, device=gpu_device)
    for L in (1, 20):
        caches = []
        for t8, s in ((k8, ks), (v8, vs)):
            t, sc = tiles.clone(), scale.clone()
            t[-4:] = t8.view(torch.uint8).to(gpu_device)
            sc[-4:] = s.to(gpu_device)
            caches.append((t, sc))
        cache = MemoryDecodeCache.__new__(MemoryDecodeCache)
        cache.num_chapters, cache.T, cache.HK, cache.dtype = C, 64, HK, FP8
        cache.k_tiles, cache.k_scale = caches[0][0].view(FP8), caches[0][1]
        from memory_amd.decode import _v8_permuted
        caches[1][0][-4:] = _v8_permuted(v8.to(gpu_device)).view(torch.uint8)
        cache.v_tiles, cache.v_scale = caches[1][0].view(FP8), caches[1][1]
        qq = q.expand(2, L, HK, 64).contiguous()
        routing = DecodeRouting((idx + C - 4).to(gpu_device), omega.to(gpu_device), C)
        qd = qq.to(gpu_device)
        got = decode_attention(qd[:, 0] if L == 1 else qd, cache, routing).view(qq.shape)
        check(got, qq, k8, ks, v8, vs, idx, omega)
        del cache, caches


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 5, 40])
def test_graph_replays(gpu_device, L):
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    q, k8, ks, v8, vs, idx, omega = make(7, L, 8, 4, 30, 9, 2)
    cache = MemoryDecodeCache.from_tiles(k8.to(gpu_device), v8.to(gpu_device), num_chapters=30, tokens_per_chapter=64,
                                         num_kv_heads=4, k_scale=ks.to(gpu_device), v_scale=vs.to(gpu_device))
    routing = DecodeRouting(idx.to(gpu_device), omega.to(gpu_device), 30)
    qd = (q[:, 0] if L == 1 else q).to(gpu_device)
    decode_attention(qd, cache, routing)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode_attention(qd, cache, routing)
    for rep in range(3):
        qd.copy_(torch.randn(qd.shape, generator=gen(rep)).to(BF))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, decode_attention(qd, cache, routing)), f"replay {rep}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(BF, 2e-2), (F32, 1e-4)])
def test_tokens_over_a_full_cache(gpu_device, dtype, tol):
    """Several query tokens over a bfloat16 or float32 cache (the sequence attention on its tiles)."""
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    q, k8, ks, v8, vs, idx, omega = make(3, 37, 8, 2, 12, 6, 4)
    idx[1, 2], idx[2, 0] = -1, 12
    k, v = (t.float() * s[:, :, None, None] for t, s in ((k8, ks), (v8, vs)))
    cache = MemoryDecodeCache.from_tiles(k.to(gpu_device, dtype), v.to(gpu_device, dtype), num_chapters=12, tokens_per_chapter=64,
                                         num_kv_heads=2)
    out = decode_attention(q.to(gpu_device), cache, DecodeRouting(idx.to(gpu_device), omega.to(gpu_device), 12))
    want, _ = reference(q, k8, ks, v8, vs, idx, omega)
    assert out.dtype == dtype and (out.cpu().double() - want).abs().max() <= tol * want.abs().max()


@pytest.mark.gpu
def test_cache_from_a_bank_saved_and_loaded(gpu_device, tmp_path):
    """The 8-bit cache of a bank is the quantised bfloat16 one; a file gives back the same bytes; a decode step and a
    prompt through it, eager and as a DecodeStepGraph."""
    from memory_amd.decode import DecodeRouting, DecodeStepGraph, MemoryDecodeCache, memory_decode_step
    from memory_amd.memory_attention import MemoryCrossAttention
    g0 = gen(3)
    C, d, H, HK, B = 9, 256, 4, 2, 5
    bank = (torch.randn(C * 64, d, generator=g0) * 0.5).to(gpu_device)
    attn = MemoryCrossAttention(d, H, HK, wo_init_zero=False).to(gpu_device, BF)
    kw = dict(num_chapters=C, tokens_per_chapter=64, num_kv_heads=HK, norm_type="rms")
    full = MemoryDecodeCache(bank, attn.k_proj.weight, attn.v_proj.weight, **kw)
    eight = MemoryDecodeCache(bank, attn.k_proj.weight, attn.v_proj.weight, dtype=FP8, **kw)
    again = full.quantized()
    same = lambda a, b: all(torch.equal(getattr(a, n).view(torch.uint8), getattr(b, n).view(torch.uint8))
                            for n in ("k_tiles", "v_tiles", "k_scale", "v_scale"))
    assert same(eight, again) and eight.nbytes < 0.51 * full.nbytes
    path = str(tmp_path / "cache.safetensors")
    eight.save(path)
    assert same(MemoryDecodeCache.load(path, gpu_device), eight)
    idx = torch.stack([torch.randperm(C, generator=g0)[:5] for _ in range(B)]).int().to(gpu_device)
    routing = DecodeRouting(idx, torch.rand(B, 5, generator=g0).to(gpu_device), C)
    k, v = eight.dequantized()
    exact = MemoryDecodeCache.from_tiles(k, v, num_chapters=C, tokens_per_chapter=64, num_kv_heads=HK)
    attn32 = MemoryCrossAttention(d, H, HK, wo_init_zero=False).to(gpu_device)
    attn32.load_state_dict({n: p.float() for n, p in attn.state_dict().items()})
    assert memory_decode_step(attn, torch.zeros(B, 0, d, device=gpu_device, dtype=BF), eight, routing).shape == (B, 0, d)
    for L in (1, 12):
        h = torch.randn(B, L, d, generator=g0).to(gpu_device, BF)
        got = memory_decode_step(attn, h, eight, routing)
        want = memory_decode_step(attn32, h.float(), exact, routing)
        # bfloat16 queries, attention and result: each 2^-8 of magnitudes that the projections mix
        assert got.shape == h.shape and (got.float() - want).abs().max() <= 2e-2 * want.abs().max()
        graph = DecodeStepGraph([(attn, eight, routing)], [h])
        for rep in range(3):
            x = torch.randn(B, L, d, generator=gen(rep)).to(gpu_device, BF)
            out = graph.run([x])[0].clone()
            torch.cuda.synchronize()
            assert torch.equal(out, memory_decode_step(attn, x, eight, routing))


@pytest.mark.gpu
def test_refusals(gpu_device):
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    k8, s = make_tiles(4, 2, 1)
    k8, s = k8.to(gpu_device), s.to(gpu_device)
    kw = dict(num_chapters=4, tokens_per_chapter=64, num_kv_heads=2)
    for bad in (dict(), dict(k_scale=s), dict(k_scale=s, v_scale=-s), dict(k_scale=s * float("inf"), v_scale=s),
                dict(k_scale=s[:, :1], v_scale=s)):
        with pytest.raises(ValueError):
            MemoryDecodeCache.from_tiles(k8, k8, **kw, **bad)
    with pytest.raises(ValueError):
        MemoryDecodeCache.from_tiles(k8.float(), k8.float(), **kw, k_scale=s, v_scale=s)
    cache = MemoryDecodeCache.from_tiles(k8, k8, **kw, k_scale=s, v_scale=s)
    idx = torch.zeros(3, 2, device=gpu_device, dtype=torch.int32)
    routing = DecodeRouting(idx, torch.ones(3, 2, device=gpu_device), 4)
    for shape in ((2, 4, 64), (3, 3, 64), (3, 4, 32), (3, 64), (3, 1, 1, 4, 64)):
        with pytest.raises(ValueError):
            decode_attention(torch.zeros(shape, device=gpu_device, dtype=BF), cache, routing)
    wide = DecodeRouting(idx, torch.ones(3, 2, device=gpu_device), 5)
    with pytest.raises(ValueError, match="cache of 4"):
        decode_attention(torch.zeros(3, 4, 64, device=gpu_device, dtype=BF), cache, wide)


def test_refusals_of_the_entry_points():
    import ctypes
    from memory_amd import _lib as L
    from memory_amd.decode import _Cache8Args, _v8_natural, _v8_permuted
    v = torch.randint(0, 255, (3, 2, 64, 64), dtype=torch.uint8, generator=gen(1)).view(FP8)
    p = _v8_permuted(v).view(torch.uint8)
    for g in range(4):
        for kb in range(4):
            for x in range(4):
                assert torch.equal(p[..., 16 * g + 4 * kb + x], v.view(torch.uint8)[..., 16 * kb + 4 * g + x, :])
    assert torch.equal(_v8_natural(_v8_permuted(v)).view(torch.uint8), v.view(torch.uint8))
    with pytest.raises(ValueError, match="null"):
        L.call("moc_cache8_pack", L.MOC_BF16, None, None, 3, None, None, None, None, None)
    with pytest.raises(ValueError, match="dtype"):
        L.call("moc_cache8_pack", 7, 16, 16, 3, 16, 16, 16, 16, None)
    ok = dict(B=1, L=1, H=2, HK=1, NS=3, C=4, max_u=3)
    for bad in (dict(), dict(H=3, HK=2), dict(NS=0), dict(L=0), dict(C=0), dict(max_u=-1), dict(B=1 << 20, L=1 << 11)):
        a = _Cache8Args(**{**ok, **bad})
        with pytest.raises(ValueError):
            L.call("moc_cache8_attend", ctypes.addressof(a), None, 0, None)
    ptrs = {n: 256 for n, t in _Cache8Args._fields_ if t is ctypes.c_void_p}
    a = _Cache8Args(**ok, **ptrs)
    with pytest.raises(ValueError, match="workspace"):
        L.call("moc_cache8_attend", ctypes.addressof(a), 256, 16, None)
    a.q = 8
    with pytest.raises(ValueError, match="aligned"):
        L.call("moc_cache8_attend", ctypes.addressof(a), 256, 1 << 20, None)


def tight(q, k8, ks, v8, vs, idx, omega):
    """(o, bound) with the bound of float16 probabilities and part rows: the result's rounding 2^-8 |o|; probabilities, row
    sums or part rows 2^-11 each and 2^-11 for everything in float32 (sums of up to 2^11 terms of 2^-24, exponentials,
    quotients) on sum_j p_j |v_j|; the logits' float32 sums, 2^-16 of the largest logit's terms; float16's smallest
    step, 2^-24 of the row's largest probability per key (in its numerator and, for the row sum, on |o|) and 2^-25 of a
    value factor for a part row."""
    B, Lq, H, D = q.shape
    C, HK = ks.shape
    out, bound = torch.zeros(B, Lq, H, D, dtype=torch.float64), torch.zeros(B, Lq, H, D, dtype=torch.float64)
    for b in range(B):
        sl = [s for s in range(idx.shape[1]) if 0 <= int(idx[b, s]) < C]
        if not sl:
            continue
        ids, om = idx[b, sl].long(), omega[b, sl].double()
        k = k8[ids].to(F32).double() * ks[ids].double()[:, :, None, None] * om[:, None, None, None]
        f = vs[ids].double() * om[:, None]                              # value factors [slots][HK]
        v = v8[ids].to(F32).double() * f[:, :, None, None]
        qd = q[b].double().transpose(0, 1).view(HK, H // HK, Lq, D)
        for hk in range(HK):
            kk, vv = k[:, hk].reshape(-1, D), v[:, hk].reshape(-1, D)
            x = qd[hk].reshape(-1, D)
            p = torch.softmax(x @ kk.t() / 8, dim=1)
            o, mag = p @ vv, p @ vv.abs()
            logit = (x.abs() @ kk.abs().t() / 8).amax(1, keepdim=True)
            top = p.amax(1, keepdim=True)
            part = p.view(p.shape[0], len(sl), 64).sum(2) @ f[:, hk, None].abs()
            e = (H8 * o.abs() + (3 * 2.0 ** -11 + 2.0 ** -16 * logit) * mag + 2.0 ** -24 * top * vv.abs().sum(0)
                 + 2.0 ** -24 * 64 * len(sl) * top * o.abs() + 2.0 ** -25 * part)
            at = slice(hk * (H // HK), (hk + 1) * (H // HK))
            out[b, :, at] = o.view(H // HK, Lq, D).transpose(0, 1)
            bound[b, :, at] = e.view(H // HK, Lq, D).transpose(0, 1)
    return out, bound


def check_tight(got, *case):
    want, bound = tight(*case)
    err = (got.cpu().double() - want).abs()
    print(f"q {tuple(case[0].shape)}: worst {(err / (bound + 1e-30)).max().item():.3f} of the bound", flush=True)
    assert (err <= bound + 1e-30).all()      # (NaN and infinity fail too)


def prompts(B, Lq, H, HK, C, NS, seed):
    """make() of a shape whose row blocks each take all slots in one workgroup (no part rows, so no workspace)."""
    from memory_amd.decode import _attend8_workspace
    assert _attend8_workspace(B, Lq, H, HK, NS) == 0
    return make(B, Lq, H, HK, C, NS, seed)


MANY = [(160, 65, 1, 1, 30, 24), (33, 130, 4, 2, 40, 17), (3, 400, 32, 8, 40, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY)
def test_prompts_of_many_slots_per_workgroup(gpu_device, shape):
    """Many slots one after the other in one workgroup: ordinary ones, skipped ids between live ones (the first and the
    last among them), zero factors in the middle, whole sequences without a slot."""
    case = list(prompts(*shape, seed=41))
    check_tight(attend(gpu_device, *case), *case)
    idx, omega, vs = case[5].clone(), case[6].clone(), case[4].clone()
    B, NS = idx.shape
    idx[torch.rand(B, NS, generator=gen(5)) < 0.3] = -1
    idx[0, 0], idx[0, -1], idx[1, 3:6] = -1, 99, -5
    idx[2] = -1
    omega[torch.rand(B, NS, generator=gen(6)) < 0.2] = 0
    vs[::5] = 0
    case[4], case[5], case[6] = vs, idx, omega
    got = attend(gpu_device, *case)
    check_tight(got, *case)
    assert not got[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY[:2])
def test_prompts_whose_logits_rise(gpu_device, shape):
    """Logits of several hundred that rise, fall or mix from slot to slot: the running maximum is raised at most slots;
    and a tile of NaN in the middle stays in the rows that read it."""
    case = list(prompts(*shape, seed=43))
    C, (B, NS) = shape[4], case[5].shape
    for order in ("rise", "fall", "mix"):
        size = {"rise": torch.linspace(0.2, 40, C), "fall": torch.linspace(40, 0.2, C), "mix": torch.rand(C, generator=gen(2)) * 40}[order]
        c = [*case]
        c[2] = case[2] * 0.3 * size[:, None]
        c[5] = case[5].sort(1).values
        check_tight(attend(gpu_device, *c), *c)
    clean = attend(gpu_device, *c)
    k8 = c[1].view(torch.uint8).clone()
    hit = int(c[5][1, NS // 2])
    k8[hit, -1, 3, 3] = 0x7f
    c[1] = k8.view(FP8)
    got = attend(gpu_device, *c)
    HK, G = shape[3], shape[2] // shape[3]
    for b in range(B):
        own = slice((HK - 1) * G, HK * G)
        assert torch.equal(got[b, :, :(HK - 1) * G], clean[b, :, :(HK - 1) * G])
        assert got[b, :, own].isnan().all() if (c[5][b] == hit).any() else torch.equal(got[b, :, own], clean[b, :, own])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MANY[:2])
@pytest.mark.parametrize("chain", [(60, -20, -80), (60, 0, -29, -60, -90, -100), (-120, -60, 0, 60, 100), (110, 30, 25, -50, -120),
                                   (-100, 60, -20, -80, 60, -29, -110), (0, -80, -125)])
@pytest.mark.parametrize("by", ["scale", "weight"])
def test_chains_of_value_factors(gpu_device, shape, chain, by):
    """Value factors that fall, rise or alternate by up to 2^80 a slot and 2^230 in all, from the scales or (to 2^-125)
    from the routing weights, in slot order: finite, and right within the factors that may count as nothing (below
    2^-90 of the largest, which are far below the bound where the probabilities are alike)."""
    if by == "weight" and max(chain) > 60:
        chain = tuple(e - max(chain) for e in chain)
    case = list(prompts(*shape, seed=47))
    q, k8, ks, v8, vs, idx, omega = case
    B, NS = idx.shape
    C = ks.shape[0]
    f = torch.exp2(torch.tensor(chain, dtype=F32).clamp(min=-125))
    per = -(-NS // len(chain))
    order = torch.arange(NS) // per
    idx = torch.stack([torch.randperm(C, generator=gen(b))[:NS] for b in range(B)]).sort(1).values.int()
    idx[:] = idx[0]                      # slots of all sequences alike, so that a chapter's scale is its slot's
    q = (q.float() * 0.1).to(BF)
    if by == "scale":
        vs = torch.ones_like(vs)
        vs[idx[0].long()] = f[order][:, None]
        omega = torch.ones_like(omega)
    else:
        vs, omega = torch.ones_like(vs), f[order].expand(B, NS).contiguous()
        omega = omega * torch.where(omega == omega.max(), 0.3, 1.0)
    case = (q, k8, ks, v8, vs, idx, omega)
    got = attend(gpu_device, *case)
    assert got.isfinite().all()
    check_tight(got, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 4, 65])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 24, 2.0 ** 40, 2.0 ** 60])
def test_logits_without_a_fraction(gpu_device, L, size):
    """Logits so large that float32 holds no fraction of them: every row is finite, and where the largest leads by more
    than their rounding (2^-16 of the largest logit's terms, and 30 for the others' probabilities) it takes all."""
    case = prompts(160, 65, 1, 1, 30, 24, 59) if L == 65 else make(16, L, 4, 2, 12, 5, 59)
    q, k8, ks, v8, vs, idx, omega = case
    omega = 0.5 + omega / 2
    ks = ks * size
    case = (q, k8, ks, v8, vs, idx, omega)
    got = attend(gpu_device, *case)
    assert got.isfinite().all()
    want, _ = reference(*case)
    B, Lq, H, _ = q.shape
    HK, rows, clear = ks.shape[1], 0, 0
    for b in range(B):
        ids, om = idx[b].long(), omega[b].double()
        for h in range(H):
            k = (k8[ids].to(F32).double() * ks[ids].double()[:, :, None, None] * om[:, None, None, None])[:, h // (H // HK)].reshape(-1, 64)
            s, terms = q[b, :, h].double() @ k.t() / 8, (q[b, :, h].double().abs() @ k.abs().t() / 8).amax(1)
            two = s.topk(2, dim=1).values
            lead = two[:, 0] - two[:, 1] > 2.0 ** -16 * terms + 30
            err = (got[b, :, h].cpu().double() - want[b, :, h]).abs()[lead]
            # half a step of the result, and of the values' float32 factors
            assert (err <= (H8 + 2.0 ** -20) * want[b, :, h].abs()[lead] + 2.0 ** -30).all()
            rows, clear = rows + Lq, clear + int(lead.sum())
    print(f"{clear} of {rows} rows are clear", flush=True)
    assert clear > rows // 2


@pytest.mark.gpu
def test_full_tiles_of_any_address(gpu_device):
    """bfloat16 and float32 tiles that start off a 16-byte boundary are copied to one when a cache is made of them."""
    from memory_amd.decode import DecodeRouting, MemoryDecodeCache, decode_attention
    q, k8, ks, v8, vs, idx, omega = make(3, 37, 4, 2, 12, 6, 4)
    kw = dict(num_chapters=12, tokens_per_chapter=64, num_kv_heads=2)
    routing = DecodeRouting(idx.to(gpu_device), omega.to(gpu_device), 12)
    for dtype in (BF, F32):
        k, v = ((t.float() * s[:, :, None, None]).to(gpu_device, dtype) for t, s in ((k8, ks), (v8, vs)))
        off = [torch.empty(t.numel() + 1, device=gpu_device, dtype=dtype)[1:].view(t.shape).copy_(t) for t in (k, v)]
        caches = [MemoryDecodeCache.from_tiles(*t, **kw) for t in ((k, v), off)]
        assert caches[0].k_tiles.data_ptr() == k.data_ptr()
        assert all(t.data_ptr() % 16 == 0 for c in caches for t in (c.k_tiles, c.v_tiles))
        for x in (q, q[:, 0]):
            a, b = (decode_attention(x.to(gpu_device), c, routing) for c in caches)
            assert torch.equal(a, b)


def half_way(L, sign):
    """Half of a chapter's keys with probabilities just below (or above) the middle of two bfloat16 values, the other
    half with 1/2 of the largest, values that cancel between the halves: roundings to bfloat16 all fall on one side."""
    case = list(make(16, L, 4, 2, 3, 1, 53))
    q, k, v = torch.zeros(16, L, 4, 64), torch.zeros(3, 2, 64, 64), torch.ones(3, 2, 64, 64)
    k[:, :, 1:33, 0:4], k[:, :, 33:, 4:8] = -1.0, -1.0
    v[:, :, 33:] = -1.0
    for at, p in ((0, 0.5 + 2.0 ** -9 + sign * 2.0 ** -13), (4, 0.5)):
        rest = -8 * math.log(p)
        for i in range(4):
            q[..., at + i] = float(torch.tensor(rest).to(BF))
            rest -= float(q[0, 0, 0, at + i])
    one = torch.ones(3, 2)
    return q.to(BF), k.to(FP8), one, v.to(FP8), one, case[5], torch.ones_like(case[6])


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 4, 24])
@pytest.mark.parametrize("sign", [-1, 1])
def test_roundings_are_float16(gpu_device, L, sign):
    """Where bfloat16 probabilities would be off by more than the bound."""
    case = half_way(L, sign)
    check_tight(attend(gpu_device, *case), *case)


def test_bound_tells_bfloat16_probabilities():
    """The same attention with probabilities rounded to bfloat16 is off by more than the bound, with float16 by less."""
    for dt, fits in ((BF, False), (torch.float16, True)):
        for sign in (-1, 1):
            q, k8, ks, v8, vs, idx, omega = half_way(1, sign)
            want, bound = tight(q, k8, ks, v8, vs, idx, omega)
            s = q[0, 0, :1].double() @ k8[int(idx[0, 0]), 0].to(F32).double().t() / 8
            p = torch.exp(s - s.amax(1, keepdim=True)).to(dt).double()
            v = v8[int(idx[0, 0]), 0].to(F32).double()
            for total in (p.sum(1, keepdim=True), torch.exp(s - s.amax(1, keepdim=True)).sum(1, keepdim=True)):
                worst = (((p @ v / total).to(BF).double() - want[0, 0, :1]).abs() / bound[0, 0, :1]).max().item()
                print(dt, sign, worst)
                assert (worst <= 1) == fits
