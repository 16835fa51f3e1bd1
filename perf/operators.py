"""Operators of the memory sublayer beside its attention, as cases that can be timed and checked.

  route   ops.router_select: softmax or sigmoid scores, a balance bias that only steers the selection,
          groups of chapters, top-k, renormalised weights; the forward, or a training step (forward and
          the gradient of the logits)
  cache   decode_attention over a MemoryDecodeCache held in 8 bits (float8_e4m3fn with one scale per
          chapter and kv head), for one token per sequence or for a prompt
  join    ops.gated_residual_norm: the norm after a block, its gate, the scaled residual and the next
          block's norm in one pass; the forward, or a training step with every gradient

``own`` says which side ``run`` takes: the plain torch form, or the framework's entry points.  Chapters
hold 64 rows, heads 64 dims, and the first chapter is shared, as everywhere in this framework.
"""

import math
import random

import torch

own = False

D = 64          # head dimension
T = 64          # rows of a chapter
SHARED = 1      # shared chapters in front
EPS = 1e-5      # of both norms


def listed():
    return [
        # routing decided again for a serving batch: one row per sequence, the whole bank, 64 chapters
        dict(name="route_step", kind="route", train=False, R=16, C=4097, k=64, score="sigmoid", bias=True, G=8, g=4,
             best=2, renorm=True, scale=1.0),
        # the tokens of one prompt (odd length), sixteen groups of which four stay
        dict(name="route_prompt", kind="route", train=False, R=2039, C=4097, k=16, score="sigmoid", bias=True, G=16,
             g=4, best=2, renorm=True, scale=2.5),
        # token-level training step at the paper's bank: 4 x 2,048 tokens
        dict(name="route_train", kind="route", train=True, R=8192, C=4097, k=16, score="sigmoid", bias=True, G=8, g=4,
             best=2, renorm=True, scale=1.0),
        # a small bank trained with softmax scores that are not renormalised: every logit has a gradient
        dict(name="route_train_softmax", kind="route", train=True, R=16001, C=257, k=8, score="softmax", bias=False,
             G=1, g=1, best=1, renorm=False, scale=1.0),
        # one user's token: 65 chapters of 12 heads, where latency counts
        dict(name="cache_one", kind="cache", B=1, L=1, H=12, HK=12, C=4097, k=64),
        # a serving batch of 64 sequences: HBM traffic of the selected chapters
        dict(name="cache_batch", kind="cache", B=64, L=1, H=12, HK=12, C=4097, k=64),
        # grouped heads, an odd batch
        dict(name="cache_grouped", kind="cache", B=37, L=1, H=16, HK=4, C=4097, k=64),
        # one prompt of odd length over the 8-bit memory
        dict(name="cache_prompt", kind="cache", B=1, L=509, H=12, HK=12, C=4097, k=64),
        # long prompts of a batch, grouped heads: matrix work
        dict(name="cache_prompts", kind="cache", B=4, L=2048, H=16, HK=4, C=4097, k=64),
        # the end of a sublayer for one token of 16 sequences
        dict(name="join_step", kind="join", train=False, R=16, d=768, x="bf16", res="bf16", norm="rms", gate="channel",
             alpha=1.0),
        # the paper's layer trained: 8 x 1,024 tokens, residual stream in float32, one gate per channel
        dict(name="join_train", kind="join", train=True, R=8192, d=768, x="bf16", res="f32", norm="rms",
             gate="channel", alpha=1.0),
        # a wide model, ragged row count, one gate per token, LayerNorm, scaled residual
        dict(name="join_train_wide", kind="join", train=True, R=6123, d=4096, x="bf16", res="bf16", norm="layer",
             gate="token", alpha=0.7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["route", "route", "cache", "cache", "join", "join"])
    if kind == "route":
        train = rng.random() < 0.5
        G = rng.choice([1, 1, 2, 4, 8, 16, 3])
        g = rng.randint(1, G)
        per = _log(rng, max(4, 32 // G), 4096 // G)
        C = SHARED + G * per
        k = min(_log(rng, 1, 64), g * per)
        score = rng.choice(["sigmoid", "sigmoid", "softmax"])
        return dict(kind=kind, train=train, R=min(_log(rng, 1, 16384), 8192 * 4097 // C), C=C, k=k, score=score,
                    bias=rng.random() < 0.7, G=G, g=g, best=min(rng.choice([1, 2, 2]), per),
                    renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))
    if kind == "cache":
        H, HK = rng.choice([(12, 12), (12, 12), (12, 4), (8, 8), (16, 4), (8, 1), (4, 2)])
        C = _log(rng, 33, 4097)
        k = min(_log(rng, 4, 64), C - 1)
        L = rng.choice([1, 1, 1, _log(rng, 2, 2048)])
        B = _log(rng, 1, 64) if L == 1 else max(1, min(_log(rng, 1, 8), 8192 // L))
        return dict(kind=kind, B=B, L=L, H=H, HK=HK, C=C, k=k)
    d = rng.choice([256, 512, 768, 768, 1024, 2048, 4096, 2 * _log(rng, 50, 1500) + 1])
    return dict(kind=kind, train=rng.random() < 0.6, R=max(1, min(_log(rng, 1, 16384), 6123 * 4096 // d)), d=d,
                x=rng.choice(["bf16", "bf16", "f32"]), res=rng.choice(["bf16", "f32"]),
                norm=rng.choice(["rms", "rms", "layer"]), gate=rng.choice(["scalar", "channel", "token", "full", "none"]),
                alpha=rng.choice([1.0, 0.7]))


# --------------------------------------------------------------------------------- inputs

def _dt(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _gen(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return torch.Generator(device=dev).manual_seed(seed), dev


def prepare(case, seed):
    return {"route": _prepare_route, "cache": _prepare_cache, "join": _prepare_join}[case["kind"]](case, seed)


def _prepare_route(case, seed):
    """Logits of hidden states N(0, 1) on router rows N(0, 0.02) at d = 768 are N(0, 0.55); a balance bias that
    has moved some way from 0."""
    g, dev = _gen(seed)
    R, C, k = case["R"], case["C"], case["k"]
    st = dict(case=case, logits=torch.randn(R, C, generator=g, device=dev) * 0.55)
    st["bias"] = torch.randn(C, generator=g, device=dev) * 0.02 if case["bias"] else None
    st["dw"] = torch.randn(R, k, generator=g, device=dev) if case["train"] else None
    if case["train"]:
        st["logits"].requires_grad_(True)
    return st


def _pow2_scale(amax):
    """The power of two that brings a tile's largest magnitude to 448 or just below."""
    return torch.exp2(torch.ceil(torch.log2(amax.double() / 448.0))).float()


def _cache_tiles(case, seed):
    """8-bit K and V tiles [C][HK][64 keys][64 dims] with their scales [C][HK], magnitudes that differ from chapter
    to chapter, queries, distinct chapters per sequence and their weights (the shared chapter's first)."""
    g, dev = _gen(seed)
    B, L, H, HK, C, k = (case[n] for n in ("B", "L", "H", "HK", "C", "k"))

    def tiles():
        x = torch.randn(C, HK, T, D, generator=g, device=dev, dtype=torch.float32)
        x *= torch.exp(0.5 * torch.randn(C, HK, 1, 1, generator=g, device=dev))
        s = _pow2_scale(x.abs().amax((2, 3)))
        x /= s[:, :, None, None]
        return x.to(torch.float8_e4m3fn), s

    k8, ks = tiles()
    v8, vs = tiles()
    q = torch.randn(B, L, H, D, generator=g, device=dev).bfloat16()
    z = torch.randn(B, C - 1, generator=g, device=dev)
    top, ids = z.topk(k, dim=1)
    w = torch.softmax(top, 1)
    omega = torch.cat([torch.ones(B, 1, device=dev), 2.5 * w], 1) / 3.5
    idx = torch.cat([torch.zeros(B, 1, device=dev, dtype=torch.int32), (ids + 1).int()], 1)
    return k8, ks, v8, vs, (q[:, 0] if L == 1 else q).contiguous(), idx, omega


def _prepare_cache(case, seed):
    k8, ks, v8, vs, q, idx, omega = _cache_tiles(case, seed)
    st = dict(case=case, q=q)
    if own:     # a server keeps the cache, and the plan of a generation's routing
        from memory_amd.decode import DecodeRouting, MemoryDecodeCache
        st["cache"] = MemoryDecodeCache.from_tiles(k8, v8, num_chapters=case["C"], tokens_per_chapter=T,
                                                   num_kv_heads=case["HK"], k_scale=ks, v_scale=vs)
        st["routing"] = DecodeRouting(idx, omega, case["C"])
    else:
        st.update(k8=k8, ks=ks, v8=v8, vs=vs, idx=idx, omega=omega)
    return st


def _prepare_join(case, seed):
    """The block's output (smaller than the stream it is added to), the residual stream, norm weights near 1,
    gates below 1, and upstream gradients of both results."""
    g, dev = _gen(seed)
    R, d = case["R"], case["d"]
    xt, rt = _dt(case["x"]), _dt(case["res"])

    def n(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)

    st = dict(case=case, x=n(R, d, std=0.3, dtype=xt), r=n(R, d, std=1.5, dtype=rt), w1=n(d, std=0.1, mean=1.0),
              w2=n(d, std=0.1, mean=1.0), b1=None, b2=None, gate=None)
    if case["norm"] == "layer":
        st.update(b1=n(d, std=0.1), b2=n(d, std=0.1))
    shape = {"none": None, "scalar": (1,), "channel": (d,), "token": (R, 1), "full": (R, d)}[case["gate"]]
    if shape is not None:
        st["gate"] = n(*shape, std=0.2, mean=0.5, dtype=torch.float32 if case["gate"] in ("scalar", "channel") else xt)
    if case["train"]:
        st.update(dh=n(R, d, dtype=rt), dn=n(R, d, dtype=xt))
        for name in ("x", "r", "w1", "w2", "b1", "b2", "gate"):
            if st[name] is not None:
                st[name].requires_grad_(True)
    return st


# --------------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"route": _own_route, "cache": _own_cache, "join": _own_join}[kind](state)
    return {"route": _plain_route, "cache": _plain_cache, "join": _plain_join}[kind](state)


def _own_route(st):
    from memory_amd import ops
    c = st["case"]
    idx, w = ops.router_select(st["logits"], c["k"], SHARED, score=c["score"], bias=st["bias"], num_groups=c["G"],
                               top_groups=c["g"], group_best=c["best"], renormalize=c["renorm"], scale=c["scale"])
    if not c["train"]:
        return idx, w
    (dz,) = torch.autograd.grad(w, st["logits"], st["dw"])
    return idx, w.detach(), dz


def _own_cache(st):
    from memory_amd.decode import decode_attention
    return decode_attention(st["q"], st["cache"], st["routing"])


def _own_join(st):
    from memory_amd import ops
    c = st["case"]
    h, n = ops.gated_residual_norm(st["x"], st["r"], post_weight=st["w1"], post_bias=st["b1"], gate=st["gate"],
                                   residual_scale=c["alpha"], pre_weight=st["w2"], pre_bias=st["b2"], eps=EPS,
                                   norm=c["norm"], out_dtype=_dt(c["x"]))
    if not c["train"]:
        return h, n
    leaves = [st[name] for name in ("x", "r", "gate", "w1", "b1", "w2", "b2") if st[name] is not None]
    return (h.detach(), n.detach(), *torch.autograd.grad([h, n], leaves, [st["dh"], st["dn"]]))


# The plain forms: elementary operations in float32, rounded once at the end.

@torch.no_grad()
def _plain_route(st):
    c = st["case"]
    z, dw = st["logits"].detach(), st["dw"]
    R, C, k, G = c["R"], c["C"], c["k"], c["G"]
    zs = z[:, SHARED:]
    # the selection in float64: neighbouring keys differ by less than float32 resolves
    z64 = zs.double()
    if c["score"] == "softmax":
        e = torch.exp(z64 - z64.amax(1, keepdim=True))
        key = e / e.sum(1, keepdim=True)
    else:
        key = 1.0 / (1.0 + torch.exp(-z64))
    if c["bias"]:
        key = key + st["bias"][SHARED:].double()
    if c["g"] < G:
        grp = key.view(R, G, -1)
        gs = grp.topk(c["best"], dim=2).values.sum(2)
        keep = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :c["g"]]
        live = torch.zeros(R, G, dtype=torch.bool, device=z.device).scatter_(1, keep, True)
        key = torch.where(live[:, :, None], grp, float("-inf")).view(R, -1)
    pos = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    # scores and weights in float32
    if c["score"] == "softmax":
        e = torch.exp(zs - zs.amax(1, keepdim=True))
        s = e / e.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-zs))
    sel = s.gather(1, pos)
    den = sel.sum(1, keepdim=True).clamp_min(1e-12)
    w = c["scale"] * (sel / den if c["renorm"] else sel)
    idx = (pos + SHARED).int()
    if not c["train"]:
        return idx, w
    ds = c["scale"] * dw
    if c["renorm"]:
        ds = (ds - (ds * sel).sum(1, keepdim=True) / den) / den
    dz = torch.zeros_like(z)
    if c["score"] == "softmax":
        dzs = -s * (ds * sel).sum(1, keepdim=True)
        dzs.scatter_add_(1, pos, ds * sel)
        dz[:, SHARED:] = dzs
    else:
        dz[:, SHARED:].scatter_(1, pos, ds * sel * (1.0 - sel))
    return idx, w, dz


@torch.no_grad()
def _plain_cache(st):
    c = st["case"]
    B, L, H, HK, NS = c["B"], c["L"], c["H"], c["HK"], c["k"] + SHARED
    idx, G = st["idx"].long(), H // HK
    om = st["omega"][:, :, None, None]
    # keys and values of each sequence's chapters, with the chapter's weight: [B][HK][NS * 64][64]
    ks, vs = st["ks"][idx][:, :, :, None, None], st["vs"][idx][:, :, :, None, None]
    K = (st["k8"].view(torch.uint8)[idx].view(torch.float8_e4m3fn).float() * ks * om[..., None]).transpose(1, 2)
    K = K.reshape(B, HK, NS * T, D)
    V = (st["v8"].view(torch.uint8)[idx].view(torch.float8_e4m3fn).float() * vs * om[..., None]).transpose(1, 2)
    V = V.reshape(B, HK, NS * T, D)
    q = st["q"].view(B, L, HK, G, D).float().permute(0, 2, 3, 1, 4).reshape(B, HK, G * L, D)
    s = torch.matmul(q, K.transpose(2, 3).contiguous()) * D ** -0.5
    p = torch.exp(s - s.amax(3, keepdim=True))
    o = torch.matmul(p, V) / p.sum(3, keepdim=True)
    o = o.view(B, HK, G, L, D).permute(0, 3, 1, 2, 4).reshape(st["q"].shape)
    return o.bfloat16()


def _plain_norm(x, w, b, kind):
    """(the norm's result, its standardised rows, 1 / deviation)"""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * rstd
    return xh * w if b is None else xh * w + b, xh, rstd


def _plain_norm_grad(dy, xh, rstd, w, kind):
    g = dy * w
    dx = g - xh * (g * xh).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - g.mean(1, keepdim=True)
    return dx * rstd


@torch.no_grad()
def _plain_join(st):
    c = st["case"]
    kind, alpha = c["norm"], c["alpha"]
    x, r = st["x"].float(), st["r"].float()
    gate = None if st["gate"] is None else st["gate"].float()
    u, xh, xr = _plain_norm(x, st["w1"], st["b1"], kind)
    h = alpha * r + (u if gate is None else gate * u)
    n, hh, hr = _plain_norm(h, st["w2"], st["b2"], kind)
    out = (h.to(st["r"].dtype), n.to(st["x"].dtype))
    if not c["train"]:
        return out
    dn = st["dn"].float()
    dh = st["dh"].float() + _plain_norm_grad(dn, hh, hr, st["w2"], kind)
    du = dh if gate is None else gate * dh
    grads = [_plain_norm_grad(du, xh, xr, st["w1"], kind).to(st["x"].dtype), (alpha * dh).to(st["r"].dtype)]
    if gate is not None:
        dg = dh * u
        dg = {"scalar": lambda: dg.sum().view(1), "channel": lambda: dg.sum(0),
              "token": lambda: dg.sum(1, keepdim=True), "full": lambda: dg}[c["gate"]]()
        grads.append(dg.to(st["gate"].dtype))
    grads.append((du * xh).sum(0))
    if st["b1"] is not None:
        grads.append(du.sum(0))
    grads.append((dn * hh).sum(0))
    if st["b2"] is not None:
        grads.append(dn.sum(0))
    return (*out, *grads)


# --------------------------------------------------------------------------------- work

def work(case):
    """Bytes of the inputs read once and the outputs written once, and the operations of one pass."""
    if case["kind"] == "route":
        R, C, k = case["R"], case["C"], case["k"]
        nbytes = R * C * 4 + (C * 4 if case["bias"] else 0) + R * k * 8
        flops = 6 * R * C
        if case["train"]:
            nbytes += R * k * 4 + R * C * 4
            flops += 4 * R * (C if case["score"] == "softmax" and not case["renorm"] else k)
        return {"bytes": nbytes, "flops": flops}
    if case["kind"] == "cache":
        B, L, H, HK, C, k = (case[n] for n in ("B", "L", "H", "HK", "C", "k"))
        # distinct chapters of B draws of k out of C - 1, and the shared one
        distinct = 1 + (C - 1) * (1.0 - (1.0 - k / (C - 1)) ** B)
        nbytes = distinct * HK * (2 * T * D + 8) + 2 * B * L * H * D * 2 + B * (k + SHARED) * 8
        return {"bytes": int(nbytes), "flops": 4 * B * L * H * (k + SHARED) * T * D}
    R, d = case["R"], case["d"]
    bx, br = (4 if case[n] == "f32" else 2 for n in ("x", "res"))
    gate = {"none": 0, "scalar": 4, "channel": 4 * d, "token": R * bx, "full": R * d * bx}[case["gate"]]
    params = (4 if case["norm"] == "layer" else 2) * 4 * d
    nbytes = 2 * R * d * (bx + br) + gate + params
    flops = 14 * R * d
    if case["train"]:   # the upstream gradients, and the gradients of both inputs, the gate and the norms
        nbytes += 2 * R * d * (bx + br) + gate + params
        flops += 30 * R * d
    return {"bytes": nbytes, "flops": flops}


# --------------------------------------------------------------------------------- exact results

def exact(case, seed):
    if case["kind"] == "route":
        return _exact_route(case, seed)
    if case["kind"] == "cache":
        return _exact_cache(case, seed)
    return _exact_join(case, seed)


def _exact_route(case, seed):
    """By ranks: a chapter's place is the number of chapters with a larger key, or an equal one and a lower id."""
    st = _prepare_route(case, seed)
    z = st["logits"].detach().double().requires_grad_(case["train"])
    body = z[:, SHARED:]
    s = torch.softmax(body, 1) if case["score"] == "softmax" else torch.sigmoid(body)
    key = s.detach()
    if case["bias"]:
        key = key + st["bias"][SHARED:].double()
    per = key.shape[1] // case["G"]
    blocks = key.unflatten(1, (case["G"], per))
    total = torch.sort(blocks, dim=2).values[:, :, per - case["best"]:].flip(2).sum(2)
    ids = torch.arange(case["G"], device=z.device)
    beats = (total[:, None, :] > total[:, :, None]) | ((total[:, None, :] == total[:, :, None])
                                                       & (ids[None, :] < ids[:, None])[None])
    out = beats.sum(2) >= case["g"]
    key = key.masked_fill(out.repeat_interleave(per, 1), -math.inf)
    order = torch.argsort(-key, dim=1, stable=True)[:, :case["k"]]
    chosen = torch.take_along_dim(s, order, 1)
    w = chosen / chosen.sum(1, keepdim=True).clamp_min(1e-12) if case["renorm"] else chosen
    w = w * case["scale"]
    idx = (order + SHARED).int()
    if not case["train"]:
        return idx, w
    (dz,) = torch.autograd.grad(w, z, st["dw"].double())
    return idx, w.detach(), dz


def _exact_cache(case, seed):
    """Sequence by sequence and kv head by kv head, chapters in their slots' order."""
    k8, ks, v8, vs, q, idx, omega = _cache_tiles(case, seed)
    B, L, H, HK = case["B"], case["L"], case["H"], case["HK"]
    out = torch.empty(B, L, H, D, device=q.device, dtype=torch.float64)
    qd = q.reshape(B, L, H, D).double()
    for b in range(B):
        sel = idx[b].tolist()
        kb = torch.stack([k8[i].double() * ks[i].double()[:, None, None] for i in sel])      # [NS][HK][64][64]
        vb = torch.stack([v8[i].double() * vs[i].double()[:, None, None] for i in sel])
        om = omega[b].double().repeat_interleave(T)
        for hk in range(HK):
            keys, vals = kb[:, hk].reshape(-1, D), vb[:, hk].reshape(-1, D) * om[:, None]
            for h in range(hk * (H // HK), (hk + 1) * (H // HK)):
                a = torch.softmax((qd[b, :, h] @ keys.t()) * om / math.sqrt(D), dim=1)
                out[b, :, h] = a @ vals
    return out.reshape(q.shape)


def _exact_join(case, seed):
    st = _prepare_join(case, seed)
    v = {n: None if st[n] is None else st[n].detach().double().requires_grad_(case["train"])
         for n in ("x", "r", "gate", "w1", "b1", "w2", "b2")}

    def norm(t, w, b):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(t, (t.shape[1],), w, b, EPS)
        return t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * w

    u = norm(v["x"], v["w1"], v["b1"])
    h = case["alpha"] * v["r"] + (u if v["gate"] is None else v["gate"] * u)
    n = norm(h, v["w2"], v["b2"])
    if not case["train"]:
        return h, n
    leaves = [v[k] for k in ("x", "r", "gate", "w1", "b1", "w2", "b2") if v[k] is not None]
    return (h.detach(), n.detach(), *torch.autograd.grad([h, n], leaves, [st["dh"].double(), st["dn"].double()]))
