"""Attention over an encoder's states and what stands around it, as cases that can be timed and checked.

  rotate  ops.qk_norm_rotate: RMS norm of every query and key head and the rotation by position, both tensors in one
          pass; the forward, or a training step with the gradients of rows and weights
  cross   ops.cross_attention: queries over keys and values of another length, ragged or masked; the forward, or a
          training step with the gradients of queries, keys and values
  page    new tokens of sequences whose keys and values lie in pages: PagedKVCache.append (norm, rotation, pages) and
          paged_attention over what the cache then holds

``own`` says which side ``run`` takes: the plain torch form, or the framework's entry points.
"""

import math
import random

import torch

own = False

EPS = 1e-6      # of the head norms
BASE = 10000.0  # of the rotation's frequencies


def listed():
    return [
        # one token of 16 sequences before its attention: the smallest call, where latency counts
        dict(name="rotate_step", kind="rotate", train=False, B=16, L=1, N=1, H=12, HK=12, D=64, R=64, dtype="bf16",
             pairs="half", weight="shared", start=1023),
        # a layer of 12 heads trained: 8 x 1,024 queries over 1,500 encoder states each
        dict(name="rotate_train", kind="rotate", train=True, B=8, L=1024, N=1500, H=12, HK=12, D=64, R=64,
             dtype="bf16", pairs="half", weight="shared", start=0),
        # wide grouped heads, half of each head rotated in interleaved pairs, a weight per head, odd lengths
        dict(name="rotate_train_wide", kind="rotate", train=True, B=4, L=2039, N=2039, H=32, HK=8, D=128, R=64,
             dtype="bf16", pairs="interleaved", weight="head", start=100000),
        # one user's token over one encoder's states
        dict(name="cross_step", kind="cross", train=False, B=1, L=1, N=1500, H=12, HK=12, D=64, dtype="bf16", mask="none"),
        # a prompt of odd length over long states, grouped heads of 128
        dict(name="cross_prompt", kind="cross", train=False, B=1, L=509, N=16001, H=16, HK=4, D=128, dtype="bf16",
             mask="none"),
        # a small configuration in float32, trained over ragged states: the whole step is small launches
        dict(name="cross_train_small_f32", kind="cross", train=True, B=4, L=128, N=333, H=4, HK=4, D=64, dtype="f32",
             mask="lengths"),
        # a layer of 12 heads trained over ragged states
        dict(name="cross_train", kind="cross", train=True, B=8, L=1024, N=1500, H=12, HK=12, D=64, dtype="bf16",
             mask="lengths"),
        # the largest: wide grouped heads, padded states with holes
        dict(name="cross_train_wide", kind="cross", train=True, B=4, L=2048, N=4097, H=32, HK=8, D=128, dtype="bf16",
             mask="keys"),
        # one user's token over a long history
        dict(name="page_one", kind="page", B=1, L=1, N=8191, H=32, HK=8, D=128, dtype="bf16", page=64),
        # a serving batch of 64 sequences of 12 heads: HBM traffic of their pages
        dict(name="page_batch", kind="page", B=64, L=1, N=4096, H=12, HK=12, D=64, dtype="bf16", page=64),
        # grouped heads, small pages, an odd batch
        dict(name="page_grouped", kind="page", B=37, L=1, N=5001, H=32, HK=8, D=128, dtype="bf16", page=16),
        # five tokens of each sequence at once (a draft being checked)
        dict(name="page_draft", kind="page", B=16, L=5, N=2047, H=16, HK=4, D=64, dtype="bf16", page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["rotate", "cross", "cross", "cross", "page", "page"])
    D = rng.choice([64, 64, 128])
    H, HK = rng.choice([(12, 12), (12, 4), (8, 8), (16, 4), (32, 8), (8, 1), (4, 2)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "rotate":
        B, L, N = _log(rng, 1, 16), _log(rng, 1, 2048), _log(rng, 1, 2048)
        rows = max(1, (4 * 2039 * 40 * 128) // (B * H * D))     # of the largest listed case
        L, N = min(L, rows // 2 + 1), min(N, rows // 2 + 1)
        return dict(kind=kind, train=rng.random() < 0.6, B=B, L=L, N=N, H=H, HK=HK, D=D,
                    R=rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), dtype=dtype,
                    pairs=rng.choice(["half", "interleaved"]), weight=rng.choice(["shared", "head", "none"]),
                    start=_log(rng, 1, 1000000))
    if kind == "cross":
        B, L, N = _log(rng, 1, 16), _log(rng, 1, 4096), _log(rng, 1, 16384)
        if dtype == "f32":
            L, N = min(L, 512), min(N, 2048)
        N = max(1, min(N, 4 * 32 * 2048 * 4097 * 2 // 3 // (B * H * L)))     # (the largest's live keys)
        return dict(kind=kind, train=rng.random() < 0.6, B=B, L=L, N=N, H=H, HK=HK, D=D, dtype=dtype,
                    mask=rng.choice(["none", "lengths", "keys"]))
    B, N = _log(rng, 1, 64), _log(rng, 8, 16384)
    N = min(N, 64 * 4096 * 12 * 64 // (B * HK * D * (2 if dtype == "f32" else 1)))
    return dict(kind=kind, B=B, L=rng.choice([1, 1, 1, rng.randint(2, 8)]), N=N, H=H, HK=HK, D=D, dtype=dtype,
                page=rng.choice([16, 32, 64, 128, 48]))


# --------------------------------------------------------------------------------- inputs

def _dt(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _gen(seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    return torch.Generator(device=dev).manual_seed(seed), dev


def _frequencies(R, dev):
    """Angle per position of each of the R / 2 pairs."""
    return torch.pow(torch.tensor(BASE, dtype=torch.float64, device=dev),
                     -torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)


def prepare(case, seed):
    return {"rotate": _prepare_rotate, "cross": _prepare_cross, "page": _prepare_page}[case["kind"]](case, seed)


def _prepare_rotate(case, seed):
    """Projected queries and keys, norm weights near 1; positions that go on from ``start``."""
    g, dev = _gen(seed)
    B, L, N, H, HK, D = (case[n] for n in ("B", "L", "N", "H", "HK", "D"))
    dt = _dt(case["dtype"])

    def n(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)

    st = dict(case=case, q=n(B, L, H, D, std=0.55), k=n(B, N, HK, D, std=0.55), wq=None, wk=None)
    if case["weight"] != "none":
        per = case["weight"] == "head"
        st.update(wq=n(*((H, D) if per else (D,)), std=0.1, mean=1.0, dtype=torch.float32),
                  wk=n(*((HK, D) if per else (D,)), std=0.1, mean=1.0, dtype=torch.float32))
    st["pq"] = case["start"] + torch.arange(L, device=dev)
    st["pk"] = case["start"] + torch.arange(N, device=dev)
    st["freq"] = _frequencies(case["R"], dev)
    if case["train"]:
        st.update(dq=n(B, L, H, D), dk=n(B, N, HK, D))
        for name in ("q", "k", "wq", "wk"):
            if st[name] is not None:
                st[name].requires_grad_(True)
    return st


def _ladder(g, dev, B, N):
    """Ragged lengths: evenly spread over (N / 2, N], in an order of the seed."""
    steps = N - (torch.arange(B, device=dev) * N) // (2 * B)
    return steps[torch.randperm(B, generator=g, device=dev)].int()


def _prepare_cross(case, seed):
    g, dev = _gen(seed)
    B, L, N, H, HK, D = (case[n] for n in ("B", "L", "N", "H", "HK", "D"))
    dt = _dt(case["dtype"])

    def n(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    st = dict(case=case, q=n(B, L, H, D), k=n(B, N, HK, D), v=n(B, N, HK, D), lengths=None, mask=None)
    if case["mask"] == "lengths":
        st["lengths"] = _ladder(g, dev, B, N)
    elif case["mask"] == "keys":      # padding behind each sequence's states, and one state in eight left out
        pos = torch.arange(N, device=dev)
        st["mask"] = (pos[None] < _ladder(g, dev, B, N)[:, None]) & (torch.rand(B, N, generator=g, device=dev) > 0.125)
    if case["train"]:
        st["do"] = n(B, L, H, D)
        for name in ("q", "k", "v"):
            st[name].requires_grad_(True)
    return st


def _page_inputs(case, seed):
    """Pages in an order of the seed, filled up to each sequence's first new token; the new tokens' projections."""
    g, dev = _gen(seed)
    B, L, N, H, HK, D, P = (case[n] for n in ("B", "L", "N", "H", "HK", "D", "page"))
    dt = _dt(case["dtype"])

    def n(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)

    first = (_ladder(g, dev, B, N) - 1).clamp_min(0)
    per = (N + L + P - 1) // P
    st = dict(case=case, q=n(B, L, H, D, std=0.55), k=n(B, L, HK, D, std=0.55), v=n(B, L, HK, D),
              wq=n(D, std=0.1, mean=1.0, dtype=torch.float32), wk=n(D, std=0.1, mean=1.0, dtype=torch.float32),
              table=torch.randperm(B * per, generator=g, device=dev).view(B, per).int(), first=first,
              freq=_frequencies(D, dev), k_pages=n(B * per, P, HK, D), v_pages=n(B * per, P, HK, D))
    st["lengths"] = first + L
    return st


def _prepare_page(case, seed):
    st = _page_inputs(case, seed)
    if own:     # a server keeps the cache and each sequence's pages and length
        from memory_amd.decode import PagedKVCache
        st["cache"] = PagedKVCache(st["k_pages"], st["v_pages"], st["table"], st["lengths"])
    return st


# --------------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "cross": _own_cross, "page": _own_page}[kind](state)
    return {"rotate": _plain_rotate, "cross": _plain_cross, "page": _plain_page}[kind](state)


def _own_rotate(st):
    from memory_amd import ops
    c = st["case"]
    q, k = ops.qk_norm_rotate(st["q"], st["k"], st["wq"], st["wk"], eps=EPS, q_positions=st["pq"], k_positions=st["pk"],
                              inv_freq=st["freq"], interleaved=c["pairs"] == "interleaved")
    if not c["train"]:
        return q, k
    leaves = [st[n] for n in ("q", "k", "wq", "wk") if st[n] is not None]
    return (q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [st["dq"], st["dk"]]))


def _own_cross(st):
    from memory_amd import ops
    o = ops.cross_attention(st["q"], st["k"], st["v"], kv_lengths=st["lengths"], key_mask=st["mask"])
    if not st["case"]["train"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, [st["q"], st["k"], st["v"]], st["do"]))


def _own_page(st):
    from memory_amd.decode import paged_attention
    cache = st["cache"]
    q = cache.append(st["k"], st["v"], positions=st["first"], q=st["q"], q_weight=st["wq"], k_weight=st["wk"], eps=EPS,
                     inv_freq=st["freq"])
    return paged_attention(q, cache, causal=True), st["k_pages"], st["v_pages"]


# The plain forms: elementary operations in float32, rounded once at the end.  Angles in float64.

def _cos_sin(pos, freq):
    a = pos.double()[..., None] * freq
    return torch.cos(a).float(), torch.sin(a).float()


def _split_pairs(x, R, pairs):
    if pairs == "half":
        return x[..., :R // 2], x[..., R // 2:R]
    return x[..., 0:R:2], x[..., 1:R:2]


def _join_pairs(a, b, rest, pairs):
    rot = torch.cat([a, b], -1) if pairs == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([rot, rest], -1)


def _plain_rotated(x, w, pos, freq, pairs):
    """(result, standardised rows, 1 / rms) of rows (B, L, H, D) in float32"""
    R = 2 * freq.shape[0]
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * rstd
    y = xh if w is None else xh * w
    cos, sin = (t.unsqueeze(-2) for t in _cos_sin(pos, freq))
    a, b = _split_pairs(y, R, pairs)
    return _join_pairs(a * cos - b * sin, b * cos + a * sin, y[..., R:], pairs), xh, rstd


def _plain_rotated_grad(dy, w, xh, rstd, pos, freq, pairs):
    R = 2 * freq.shape[0]
    cos, sin = (t.unsqueeze(-2) for t in _cos_sin(pos, freq))
    a, b = _split_pairs(dy, R, pairs)
    du = _join_pairs(a * cos + b * sin, b * cos - a * sin, dy[..., R:], pairs)
    g = du if w is None else du * w
    dx = (g - xh * (g * xh).mean(-1, keepdim=True)) * rstd
    if w is None:
        return dx, None
    dw = (du * xh).flatten(0, 1)
    return dx, dw.sum(0) if w.dim() == 2 else dw.sum((0, 1))


@torch.no_grad()
def _plain_rotate(st):
    c = st["case"]
    rows, grads, weights = [], [], []
    for x, w, p, d in (("q", "wq", "pq", "dq"), ("k", "wk", "pk", "dk")):
        y, xh, rstd = _plain_rotated(st[x].float(), st[w], st[p], st["freq"], c["pairs"])
        rows.append(y.to(st[x].dtype))
        if c["train"]:
            dx, dw = _plain_rotated_grad(st[d].float(), st[w], xh, rstd, st[p], st["freq"], c["pairs"])
            grads.append(dx.to(st[x].dtype))
            if dw is not None:
                weights.append(dw)
    return (*rows, *grads, *weights)


def _heads_first(x):
    return x.float().transpose(1, 2).contiguous()       # (B, heads, rows, D)


def _plain_softmax(q, k, live):
    """Scaled logits' softmax over the live keys, 0 in rows without any; q (B, HK, rows, D), k (B, HK, N, D)."""
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
    if live is None:
        p = torch.exp(s - s.amax(-1, keepdim=True))
        return p / p.sum(-1, keepdim=True)
    s = torch.where(live, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _live_keys(st):
    """(B, N) truth values of the keys that count, or None"""
    if st["mask"] is not None:
        return st["mask"]
    if st["lengths"] is None:
        return None
    return torch.arange(st["k"].shape[1], device=st["k"].device)[None] < st["lengths"][:, None]


def _grouped(x, HK):
    """(B, L, H, D) -> (B, HK, G * L, D)"""
    B, L, H, D = x.shape
    return x.float().view(B, L, HK, H // HK, D).permute(0, 2, 3, 1, 4).reshape(B, HK, H // HK * L, D)


def _ungrouped(x, L):
    B, HK, GL, D = x.shape
    return x.view(B, HK, GL // L, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, GL // L * HK, D)


@torch.no_grad()
def _plain_cross(st):
    c = st["case"]
    L, HK, D = c["L"], c["HK"], c["D"]
    dt = st["q"].dtype
    live = _live_keys(st)
    live = None if live is None else live[:, None, None, :]
    q, k, v = _grouped(st["q"], HK), _heads_first(st["k"]), _heads_first(st["v"])
    p = _plain_softmax(q, k, live)
    o = torch.matmul(p, v)
    out = _ungrouped(o, L).to(dt)
    if not c["train"]:
        return out
    do = _grouped(st["do"], HK)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (ds - (do * o).sum(-1, keepdim=True)) * D ** -0.5
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    return (out, _ungrouped(dq, L).to(dt), dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt))


@torch.no_grad()
def _plain_page(st):
    c = st["case"]
    B, L, HK, P = c["B"], c["L"], c["HK"], c["page"]
    dt = st["q"].dtype
    pos = st["first"].long()[:, None] + torch.arange(L, device=st["q"].device)
    q = _plain_rotated(st["q"].float(), st["wq"], pos, st["freq"], "half")[0].to(dt)
    k = _plain_rotated(st["k"].float(), st["wk"], pos, st["freq"], "half")[0].to(dt)
    page = torch.take_along_dim(st["table"].long(), pos // P, 1)
    st["k_pages"][page, pos % P] = k
    st["v_pages"][page, pos % P] = st["v"]
    table = st["table"].long()
    keys = st["k_pages"][table].flatten(1, 2)           # (B, pages * P, HK, D)
    vals = st["v_pages"][table].flatten(1, 2)
    at = torch.arange(keys.shape[1], device=keys.device)
    live = at <= pos[..., None]                         # (B, L, keys)
    live = live[:, None, None].expand(B, 1, c["H"] // HK, L, -1).flatten(2, 3)
    p = _plain_softmax(_grouped(q, HK), _heads_first(keys), live)
    # (a page's rows behind its sequence's last token hold whatever was there)
    vals = torch.where((at < st["lengths"][:, None])[..., None, None], vals, 0)
    return _ungrouped(torch.matmul(p, _heads_first(vals)), L).to(dt), st["k_pages"], st["v_pages"]


# --------------------------------------------------------------------------------- work

def _keys(case):
    """Keys of the whole batch that count."""
    B, N = case["B"], case["N"]
    if case["kind"] == "cross" and case["mask"] == "none":
        return B * N
    n = sum(N - (b * N) // (2 * B) for b in range(B))
    return n * 7 // 8 if case.get("mask") == "keys" else n


def work(case):
    """Bytes of the inputs read once and the outputs written once, and the operations of one pass."""
    B, L, N, H, HK, D = (case[n] for n in ("B", "L", "N", "H", "HK", "D"))
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rotate":
        rows = B * (L * H + N * HK)
        weights = {"none": 0, "shared": 2 * D, "head": (H + HK) * D}[case["weight"]] * 4
        nbytes = 2 * rows * D * es + 8 * (L + N) + 4 * case["R"] + weights
        flops = rows * (4 * D + 3 * case["R"])
        if case["train"]:       # the upstream gradients, and the gradients of rows and weights
            nbytes += 2 * rows * D * es + weights
            flops += rows * (9 * D + 3 * case["R"])
        return {"bytes": nbytes, "flops": flops}
    live = _keys(case)
    if case["kind"] == "cross":
        nbytes = 2 * B * L * H * D * es + 2 * live * HK * D * es + (B * N if case["mask"] == "keys" else 4 * B)
        flops = 4 * live * L * H * D
        if case["train"]:       # dO read; dQ, dK, dV written whole; the logits' and four more products
            nbytes += 2 * B * L * H * D * es + 2 * B * N * HK * D * es
            flops += 10 * live * L * H * D
        return {"bytes": nbytes, "flops": flops}
    nbytes = 2 * live * HK * D * es + B * L * (2 * H + 4 * HK) * D * es + 8 * B + 4 * (live // case["page"])
    return {"bytes": nbytes, "flops": 4 * live * L * H * D}


# --------------------------------------------------------------------------------- exact results

def exact(case, seed):
    return {"rotate": _exact_rotate, "cross": _exact_cross, "page": _exact_page}[case["kind"]](case, seed)


def _exact_rows(x, w, pos, freq, pairs):
    """The rotation as a complex product, in float64; pos has the shape of x's leading dims (B, L)."""
    R = 2 * freq.shape[0]
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    if w is not None:
        y = y * w
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos.double()[..., None, None] * freq)
    if pairs == "half":
        z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
        return torch.cat([z.real, z.imag, y[..., R:]], -1)
    z = torch.view_as_complex(y[..., :R].unflatten(-1, (-1, 2)).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), y[..., R:]], -1)


def _exact_rotate(case, seed):
    st = _prepare_rotate(case, seed)
    v = {n: None if st[n] is None else st[n].detach().double().requires_grad_(case["train"])
         for n in ("q", "k", "wq", "wk")}
    q = _exact_rows(v["q"], v["wq"], st["pq"], st["freq"], case["pairs"])
    k = _exact_rows(v["k"], v["wk"], st["pk"], st["freq"], case["pairs"])
    if not case["train"]:
        return q, k
    leaves = [v[n] for n in ("q", "k", "wq", "wk") if v[n] is not None]
    return (q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [st["dq"].double(), st["dk"].double()]))


def _attend(q, k, v, limit=None):
    """One sequence and head in float64: q (L, D) over the keys k (n, D); row i over the first limit[i]."""
    s = q @ k.t() / math.sqrt(q.shape[1])
    if limit is not None:
        s = s.masked_fill(torch.arange(k.shape[0], device=k.device) >= limit[:, None], -math.inf)
    return torch.softmax(s, 1) @ v


def _exact_cross(case, seed):
    """Sequence by sequence and head by head over the keys that count alone."""
    st = _prepare_cross(case, seed)
    B, H, G, train = case["B"], case["H"], case["H"] // case["HK"], case["train"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        if st["mask"] is not None:
            rows = st["mask"][b].nonzero().view(-1)
        else:
            rows = torch.arange(case["N"] if st["lengths"] is None else int(st["lengths"][b]), device=q.device)
        if rows.numel() == 0:
            continue
        for h in range(H):
            leaves = [t.requires_grad_(train) for t in (q[b, :, h].clone(), k[b, rows, h // G], v[b, rows, h // G])]
            o = _attend(*leaves)
            out[b, :, h] = o.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(o, leaves, st["do"][b, :, h].double())
                dq[b, :, h] = gq
                dk[b, rows, h // G] += gk
                dv[b, rows, h // G] += gv
    return (out, dq, dk, dv) if train else out


def _exact_page(case, seed):
    """The result over the pages as they stand and the new rows in float64; the pages themselves are what the plain
    form writes, rounded, and have no value of their own but in the new rows."""
    st = _page_inputs(case, seed)
    B, L, H, P = case["B"], case["L"], case["H"], case["page"]
    G = H // case["HK"]
    pos = st["first"].long()[:, None] + torch.arange(L, device=st["q"].device)
    q = _exact_rows(st["q"].double(), st["wq"].double(), pos, st["freq"], "half")
    knew = _exact_rows(st["k"].double(), st["wk"].double(), pos, st["freq"], "half")
    out = torch.empty_like(q)
    for b in range(B):
        n = int(st["lengths"][b])
        ids = st["table"][b, :(n + P - 1) // P].long()
        keys = torch.cat([st["k_pages"][ids].flatten(0, 1)[:n - L].double(), knew[b]])
        vals = torch.cat([st["v_pages"][ids].flatten(0, 1)[:n - L].double(), st["v"][b].double()])
        for h in range(H):
            out[b, :, h] = _attend(q[b, :, h], keys[:, h // G], vals[:, h // G], pos[b] + 1)
    return out, None, None
