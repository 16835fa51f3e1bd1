"""Single-token decode through sequence-routed memory layers.

For generation with the chapters and weights fixed by the prompt (the decode
use of memory_transformer/model.py:612-692 through
MemoryCrossAttention.forward with L = 1), the K/V projection of every chapter
is computed once per layer (``MemoryDecodeCache``, 0.8 GB per layer at the
paper shape) and each step only reads the tiles of the selected chapters:
q = q_proj(h_t) -> chapter-centric partial attention (each selected tile read
once per step for all sequences that chose it) -> joint merge over the
sequence's slots -> o_proj.  Inference only (no autograd).
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib as L
from . import ops
from ._lib import call, ptr, stream_ptr


FP8 = torch.float8_e4m3fn
# position -> key of a V tile's dim in 8 bits (its own inverse): the key order of the attention's probabilities
_V8_KEYS = [16 * kb + 4 * g + x for g in range(4) for kb in range(4) for x in range(4)]


def _v8_permuted(v: torch.Tensor) -> torch.Tensor:
    """[..., keys, dims] -> [..., dims, positions], or back."""
    keys = torch.tensor(_V8_KEYS, device=v.device)
    return v.view(torch.uint8).transpose(-1, -2)[..., keys].contiguous().view(FP8)


def _v8_natural(v: torch.Tensor) -> torch.Tensor:
    keys = torch.tensor(_V8_KEYS, device=v.device)
    return v.view(torch.uint8)[..., keys].transpose(-1, -2).contiguous().view(FP8)


class MemoryDecodeCache:
    """Per-layer K and V tiles [C][HK][64 keys][64 dims] of the whole bank (optionally row-normalised).

    ``dtype=torch.float8_e4m3fn`` (or ``quantized()`` of a float32 / bfloat16 cache) holds them in 8 bits: half the
    memory and half the bytes of a step.  Each (chapter, kv head) has a float32 scale for K and one for V
    (``k_scale``, ``v_scale`` [C][HK], powers of two), a value is scale times its e4m3 value, and ``v_tiles`` is then
    held as [C][HK][64 dims][64 positions] in the order the kernels read (``dequantized()`` gives both back as
    [keys][dims]).  A bank's 8-bit cache is that of its bfloat16 projection: rounded by 2^-8 there, by 2^-4 here."""

    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def __init__(self, bank: torch.Tensor, wk: torch.Tensor, wv: torch.Tensor, *, num_chapters: int,
                 tokens_per_chapter: int, num_kv_heads: int, norm_type: Optional[str] = None, eps: float = 1e-6,
                 dtype: torch.dtype = torch.bfloat16):
        L.require_gpu(bank, wk, wv)
        C, T = int(num_chapters), int(tokens_per_chapter)
        self.num_chapters, self.T, self.HK, self.dtype = C, T, int(num_kv_heads), dtype
        if dtype == FP8:
            full = MemoryDecodeCache(bank, wk, wv, num_chapters=C, tokens_per_chapter=T, num_kv_heads=num_kv_heads,
                                     norm_type=norm_type, eps=eps)
            self._pack(full)
            return
        with torch.no_grad():
            plan = ops.identity_plan(C, bank.device)
            code = ops.norm_code(norm_type)
            mean = rstd = None
            if code:
                mean, rstd = ops.row_stats(bank.contiguous(), plan, T, code, eps)
            wkv = torch.cat([wk, wv], 0).to(dtype).contiguous()
            self.k_tiles, self.v_tiles = ops.kv_project(bank.contiguous(), plan, T, wkv, self.HK, 64, mean, rstd,
                                                        dtype, ("k", "v"))

    def _pack(self, full: "MemoryDecodeCache") -> None:
        if full.T != 64:
            raise ValueError(f"an 8-bit decode cache needs 64 tokens per chapter, got {full.T}")
        shape, dev = full.k_tiles.shape, full.k_tiles.device
        self.k_tiles = torch.empty(shape, device=dev, dtype=FP8)
        self.v_tiles = torch.empty(shape, device=dev, dtype=FP8)
        self.k_scale = torch.empty(shape[:2], device=dev, dtype=torch.float32)
        self.v_scale = torch.empty(shape[:2], device=dev, dtype=torch.float32)
        with L.on_device(dev):
            call("moc_cache8_pack", L.dtype_code(full.dtype), ptr(full.k_tiles), ptr(full.v_tiles), shape[0] * shape[1],
                 ptr(self.k_tiles), ptr(self.v_tiles), ptr(self.k_scale), ptr(self.v_scale), stream_ptr(dev))

    def quantized(self) -> "MemoryDecodeCache":
        """This cache in 8 bits: per (chapter, kv head) the scale is the smallest power of two that brings the tile's
        largest finite magnitude to 448 or below; infinities become +-448 times it."""
        if self.dtype == FP8:
            return self
        out = MemoryDecodeCache.__new__(MemoryDecodeCache)
        out.num_chapters, out.T, out.HK, out.dtype = self.num_chapters, self.T, self.HK, FP8
        out._pack(self)
        return out

    def dequantized(self):
        """(K, V) float32 [C][HK][64 keys][64 dims] that the cache stands for."""
        if self.dtype != FP8:
            return self.k_tiles.float(), self.v_tiles.float()
        return (self.k_tiles.float() * self.k_scale[:, :, None, None],
                _v8_natural(self.v_tiles).float() * self.v_scale[:, :, None, None])

    @property
    def nbytes(self) -> int:
        scales = 0 if self.k_scale is None else 8 * self.k_scale.numel()
        return self.k_tiles.numel() * self.k_tiles.element_size() * 2 + scales

    # File format of a saved cache (safetensors): tensors ``k_tiles`` and ``v_tiles``, each
    # [num_chapters][num_kv_heads][tokens_per_chapter keys][64 dims] in the cache dtype (the
    # projected, optionally row-normalised bank, K = norm(M) Wk^T and V = norm(M) Wv^T per
    # chapter), and string metadata: format, num_chapters, tokens_per_chapter, num_kv_heads,
    # dtype.  The K/V of one memory layer; omega is applied at attention time.  An 8-bit cache is
    # written under a format of its own, with its scales ``k_scale`` and ``v_scale`` [num_chapters][num_kv_heads]
    # (float32) and both tiles as [keys][dims].
    FORMAT = "moc-decode-kv/1"
    FORMAT_8BIT = "moc-decode-kv-e4m3/1"

    def save(self, path: str) -> None:
        from safetensors.torch import save_file
        eight = self.dtype == FP8
        meta = {"format": self.FORMAT_8BIT if eight else self.FORMAT, "num_chapters": str(self.num_chapters), "tokens_per_chapter": str(self.T),
                "num_kv_heads": str(self.HK), "dtype": str(self.dtype).replace("torch.", "")}
        tensors = {"k_tiles": self.k_tiles.contiguous().cpu(),
                   "v_tiles": (_v8_natural(self.v_tiles) if eight else self.v_tiles.contiguous()).cpu()}
        if eight:
            tensors.update(k_scale=self.k_scale.cpu(), v_scale=self.v_scale.cpu())
        save_file(tensors, path, metadata=meta)

    @classmethod
    def load(cls, path: str, device: torch.device) -> "MemoryDecodeCache":
        from safetensors import safe_open
        with safe_open(path, framework="pt", device="cpu") as f:
            meta = f.metadata() or {}
            if meta.get("format") not in (cls.FORMAT, cls.FORMAT_8BIT):
                raise ValueError(f"{path}: not a {cls.FORMAT} or {cls.FORMAT_8BIT} decode cache (format "
                                 f"{meta.get('format')!r})")
            k, v = f.get_tensor("k_tiles"), f.get_tensor("v_tiles")
            scales = {}
            if meta["format"] == cls.FORMAT_8BIT:
                scales = {n: f.get_tensor(n).to(device) for n in ("k_scale", "v_scale")}
        C, T, HK = int(meta["num_chapters"]), int(meta["tokens_per_chapter"]), int(meta["num_kv_heads"])
        if tuple(k.shape) != (C, HK, T, 64) or k.shape != v.shape:
            raise ValueError(f"{path}: tile shape {tuple(k.shape)} does not match the metadata")
        return cls.from_tiles(k.to(device), v.to(device), num_chapters=C, tokens_per_chapter=T, num_kv_heads=HK, **scales)

    @classmethod
    def from_tiles(cls, k_tiles: torch.Tensor, v_tiles: torch.Tensor, *, num_chapters: int, tokens_per_chapter: int,
                   num_kv_heads: int, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None) -> "MemoryDecodeCache":
        """A cache over already projected tiles [num_chapters][num_kv_heads][T][64] (keys, dims).  Tiles in
        float8_e4m3fn come with their scales [num_chapters][num_kv_heads], finite and not negative (checked here, which
        waits for the stream)."""
        L.require_same_gpu(k_tiles, v_tiles, k_scale, v_scale)
        eight = k_tiles.dtype == FP8
        if k_tiles.dtype not in (torch.float32, torch.bfloat16, FP8) or v_tiles.dtype != k_tiles.dtype:
            raise ValueError("decode cache tiles must be float32, bfloat16 or float8_e4m3fn, both of one dtype")
        if eight != (k_scale is not None) or eight != (v_scale is not None):
            raise ValueError("float8_e4m3fn tiles need k_scale and v_scale, others take none")
        if k_tiles.shape != (num_chapters, num_kv_heads, tokens_per_chapter, 64) or v_tiles.shape != k_tiles.shape:
            raise ValueError(f"tiles of shape {tuple(k_tiles.shape)}, expected "
                             f"{(num_chapters, num_kv_heads, tokens_per_chapter, 64)}")
        self = cls.__new__(cls)
        self.num_chapters, self.T, self.HK, self.dtype = int(num_chapters), int(tokens_per_chapter), \
            int(num_kv_heads), k_tiles.dtype
        if not eight:
            # (the attention over several tokens copies 16-byte pieces of them to LDS)
            self.k_tiles, self.v_tiles = _aligned(k_tiles), _aligned(v_tiles)
            return self
        if self.T != 64:
            raise ValueError(f"an 8-bit decode cache needs 64 tokens per chapter, got {self.T}")
        self.k_tiles, self.v_tiles = _aligned(k_tiles), _v8_permuted(v_tiles)
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            s = s.float().contiguous()
            if s.shape != (self.num_chapters, self.HK) or not bool((s.isfinite() & (s >= 0)).all()):
                raise ValueError(f"{name}: finite scales >= 0 of shape {(self.num_chapters, self.HK)}, got "
                                 f"{tuple(s.shape)}")
            setattr(self, name, s)
        return self


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t if t.is_contiguous() else t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class DecodeRouting:
    """(chapter ids incl. the shared prefix, omega) of a batch of sequences and their plan.

    ``sync=True`` (routing fixed for a whole generation): the distinct-chapter count is read
    once (one synchronisation here, none per step), so each step launches exactly one wave per
    selected (chapter, kv head) tile.  ``sync=False`` (routing that changes every step,
    ``DecodeRouter``): no host read; the launches are sized for min(B * NS, C) chapters and the
    kernels read the count on the device (waves past it exit at once)."""

    def __init__(self, chapter_indices: torch.Tensor, chapter_weights: torch.Tensor, num_chapters: int,
                 sync: bool = True):
        L.require_gpu(chapter_indices, chapter_weights)
        self.idx = chapter_indices.to(torch.int32).contiguous()
        self.omega = chapter_weights.float().contiguous()
        self.B, self.NS = self.idx.shape
        self.plan = ops.chapter_plan(self.idx, num_chapters)
        self._n_unique = int(self.plan.n_uniq[0].item()) if sync else None
        self.max_units = self._n_unique if sync else min(self.B * self.NS, int(num_chapters))
        # the first 16 edges of every distinct chapter, read by the decode kernel with its plan
        # entries (instead of after them, through csr_off); -1 rows past the count
        self.row_tab = torch.empty(max(self.max_units, 1) * 16, device=self.idx.device, dtype=torch.int32)
        call("moc_decode_row_table", ptr(self.plan.n_uniq), ptr(self.plan.csr_off), ptr(self.plan.csr_edge),
             self.max_units, ptr(self.row_tab), stream_ptr(self.idx.device))

    @classmethod
    def _decided(cls, pooled, router, num_chapters: int, num_shared: int, top_k: int, scale: float):
        """(routing, logits) of pooled rows (B, d) f32: router linear, top-k with the shared prefix, plan and
        row table in one host call (moc_decode_route), equal to the separate ones."""
        B, d = pooled.shape
        C, S, k = int(num_chapters), int(num_shared), int(top_k)
        NS = S + k
        E = B * NS
        max_u = min(E, C)
        dev = pooled.device
        W = router.weight.contiguous()
        bias = None if router.bias is None else router.bias.float().contiguous()
        ws_bytes = L.query("moc_chapter_plan_workspace", E, C)
        logits = torch.empty(B, C, device=dev, dtype=torch.float32)
        w, omega = torch.empty(B * (k + NS), device=dev, dtype=torch.float32).split((B * k, E))
        sizes = (ws_bytes // 4, max_u, 2, E, max_u + 1, E, 16 * max_u, E, B * k)
        ws, uniq, n_uniq, edge_u, csr_off, csr_edge, row_tab, idx_star, idx = torch.empty(
            sum(sizes), device=dev, dtype=torch.int32).split(sizes)
        call("moc_decode_route", ptr(pooled), B, d, ptr(W), L.dtype_code(W.dtype), ptr(bias), C, S, k, scale, ptr(logits),
             ptr(idx), ptr(w), ptr(idx_star), ptr(omega), ptr(ws), ws_bytes, ptr(uniq), ptr(n_uniq), ptr(edge_u),
             ptr(csr_off), ptr(csr_edge), max_u, ptr(row_tab), stream_ptr(dev))
        self = cls.__new__(cls)
        self.idx, self.omega = idx_star.view(B, NS), omega.view(B, NS)
        self.B, self.NS = B, NS
        self.plan = ops.ChapterPlan(uniq, n_uniq, edge_u, csr_off, csr_edge, max_u, C)
        self._n_unique, self.max_units, self.row_tab = None, max_u, row_tab
        return self, logits

    def unique_chapters(self) -> int:
        if self._n_unique is None:
            self._n_unique = int(self.plan.n_uniq[0].item())
        return self._n_unique


def _masked_mean(states: torch.Tensor, mask: Optional[torch.Tensor]) -> torch.Tensor:
    """Mean over the sequence ignoring padding (mask == 0), the mask's rightmost positions
    aligned with the states (memory_transformer/model.py:468-493); fp32 result."""
    if mask is None:
        return ops.router_pool(states)
    if mask.dim() != 2:
        raise ValueError(f"attention_mask must be 2D (got shape {tuple(mask.shape)})")
    if mask.shape[0] != states.shape[0]:
        raise ValueError(f"attention_mask batch ({mask.shape[0]}) must match states batch ({states.shape[0]})")
    if mask.shape[1] < states.shape[1]:
        raise ValueError(f"attention_mask length ({mask.shape[1]}) must be >= states length ({states.shape[1]})")
    if mask.shape[1] != states.shape[1]:
        mask = mask[:, -states.shape[1]:]
    m = mask.to(device=states.device, dtype=torch.float32).unsqueeze(-1)
    return (states.float() * m).sum(dim=1) / m.sum(dim=1).clamp(min=1.0)


def _window_native(old: torch.Tensor, h: torch.Tensor) -> bool:
    """Whether moc_window_pool takes the window and the new states (packed rows of one type, 16-byte aligned,
    any batch stride)."""
    d = h.shape[-1]
    return (h.dim() == 3 and h.shape[1] > 0 and old.shape[1] > 0 and old.shape[0] == h.shape[0] and 0 < h.shape[0] < 65536
            and old.shape[2] == d and d % 8 == 0 and h.dtype == old.dtype and h.dtype in (torch.float32, torch.bfloat16)
            and h.device == old.device and all(
                t.stride(2) == 1 and (t.stride(1) == d or t.shape[1] == 1) and t.stride(0) % 8 == 0
                and t.data_ptr() % 16 == 0 for t in (old, h)))


class DecodeRouter:
    """Chapter routing of one memory layer during generation, re-decided at every step
    (MemoryTransformer.forward's inference strategies, memory_transformer/model.py:609-661):

      * "sequence" / "sequence-rolling": the router on the call's own hidden states (the prompt at
        prefill, the new token at each step), pooled as ChapterRouter pools them (mean, or the
        rolling-window mean of router.py:158-195);
      * "rolling": a window of the last ``window_size`` hidden states (prompt included), mean-pooled
        (padding masked) at prefill and at every step;
      * "hybrid": the prompt's full mean at prefill (its last ``window_size`` states start the
        window), then the rolling window at every step.

    Each call returns a ``DecodeRouting`` (shared chapters prepended, routed weights scaled and
    renormalised as model.py:356-391) built without a host synchronisation, for
    ``memory_decode_step``.  ``last_logits`` keeps the router logits of the last decision (fp32)."""

    STRATEGIES = ("sequence", "sequence-rolling", "sequence_rolling", "rolling", "hybrid")

    def __init__(self, router, *, num_chapters: int, num_shared_chapters: int = 1,
                 routed_scaling_factor: float = 2.5, strategy: str = "sequence", window_size: int = 128):
        if strategy not in self.STRATEGIES:
            raise ValueError(f"Unknown routing_strategy_inference: {strategy}")
        if int(window_size) <= 0:
            raise ValueError(f"routing_window_size must be > 0, got {window_size}")
        self.router = router
        self.num_chapters = int(num_chapters)
        self.num_shared = max(0, min(int(num_shared_chapters), self.num_chapters))
        self.routed_scale = float(routed_scaling_factor)
        self.strategy = strategy
        self.window = int(window_size)
        self.cache: Optional[torch.Tensor] = None   # (B, <= window, d): the rolling window
        self.last_logits: Optional[torch.Tensor] = None

    def reset(self) -> None:
        self.cache = None
        self.last_logits = None

    def _decide(self, pooled: torch.Tensor) -> DecodeRouting:
        from .model import prepend_shared_chapters32
        r = self.router.router
        C, S = self.num_chapters, self.num_shared
        k = min(int(self.router.top_k), C - S)
        plain = getattr(self.router, "plain_selection", True)
        if (plain and S > 0 and k > 0 and pooled.shape[0] > 0 and pooled.dtype == torch.float32 and pooled.is_contiguous()
                and r.weight.dtype in (torch.float32, torch.bfloat16) and r.weight.shape == (C, pooled.shape[1])
                and r.weight.is_cuda and (r.bias is None or r.bias.is_cuda) and L.KERNEL_EVENTS is None):
            routing, self.last_logits = DecodeRouting._decided(pooled, r, C, S, k, self.routed_scale)
            return routing
        logits = ops.router_linear(pooled, r.weight, r.bias)
        self.last_logits = logits
        if k > 0:
            idx, w = ops.router_topk(logits, k, S) if plain else self.router.select(logits, k, S)
        else:
            idx = torch.empty((pooled.shape[0], 0), dtype=torch.int32, device=pooled.device)
            w = torch.empty((pooled.shape[0], 0), dtype=torch.float32, device=pooled.device)
        idx_star, omega = prepend_shared_chapters32(idx, w, num_chapters=C, num_shared_chapters=S,
                                                    routed_scaling_factor=self.routed_scale)
        return DecodeRouting(idx_star, omega, C, sync=False)

    def _own_states(self, hidden_states: torch.Tensor) -> torch.Tensor:
        if self.strategy == "sequence":
            return ops.router_pool(hidden_states)
        from .router import rolling_coefficients
        coef = rolling_coefficients(hidden_states.shape[1], self.window, hidden_states.device)
        return ops.router_pool(hidden_states, coef)

    def _window(self, hidden_states: torch.Tensor, attention_mask: Optional[torch.Tensor]) -> torch.Tensor:
        if self.cache is not None and attention_mask is None and _window_native(self.cache, hidden_states):
            return self._advance(hidden_states)
        combined = hidden_states if self.cache is None else torch.cat([self.cache, hidden_states], dim=1)
        if combined.shape[1] > self.window:
            combined = combined[:, -self.window:]
        self.cache = combined.detach()
        return _masked_mean(combined, attention_mask)

    def _advance(self, hidden_states: torch.Tensor) -> torch.Tensor:
        """The window moved on by the new states and its mean, in one pass (moc_window_pool)."""
        old, h = self.cache, hidden_states
        B, n_old, d = old.shape
        n_new = h.shape[1]
        n = min(n_old + n_new, self.window)
        out = torch.empty(B, n, d, device=h.device, dtype=h.dtype)
        ws_bytes = L.query("moc_router_pool_workspace", B, n, d)
        pooled = torch.empty(B * d + ws_bytes // 4, device=h.device, dtype=torch.float32)
        call("moc_window_pool", ptr(old), old.stride(0), n_old, ptr(h), h.stride(0), n_new, L.dtype_code(h.dtype), B, n, d,
             ptr(out), ptr(pooled), pooled.data_ptr() + 4 * B * d, ws_bytes, stream_ptr(h.device))
        self.cache = out
        return pooled[:B * d].view(B, d)

    @torch.no_grad()
    def prefill(self, hidden_states: torch.Tensor, attention_mask: Optional[torch.Tensor] = None) -> DecodeRouting:
        """Routing of the prompt (B, P, d); starts a new window."""
        L.require_gpu(hidden_states)
        self.reset()
        if self.strategy == "hybrid":
            pooled = _masked_mean(hidden_states, attention_mask)
            self.cache = hidden_states[:, -self.window:].detach()
            return self._decide(pooled)
        if self.strategy == "rolling":
            return self._decide(self._window(hidden_states, attention_mask))
        return self._decide(self._own_states(hidden_states))

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, attention_mask: Optional[torch.Tensor] = None) -> DecodeRouting:
        """Routing of one generated token's hidden states (B, 1, d)."""
        L.require_gpu(hidden_states)
        if self.strategy in ("rolling", "hybrid"):
            return self._decide(self._window(hidden_states, attention_mask))
        return self._decide(self._own_states(hidden_states))


class _Cache8Args(ctypes.Structure):
    """moc_cache8_args."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k_tiles", "v_tiles", "k_scale", "v_scale", "omega", "idx", "uniq",
                                                "n_uniq", "csr_off", "csr_edge", "edge_u", "row_tab", "out")]
                + [(n, ctypes.c_int64) for n in ("max_u", "B", "L", "C")]
                + [(n, ctypes.c_int) for n in ("H", "HK", "NS")] + [("scale", ctypes.c_float)])


_pack_cache8 = L.packer(_Cache8Args)


@functools.lru_cache(maxsize=1024)
def _attend8_workspace(B: int, Lq: int, H: int, HK: int, NS: int) -> int:
    return L.query("moc_cache8_attend_workspace", B, Lq, H, HK, NS)


def _attend8(q: torch.Tensor, B: int, Lq: int, H: int, cache: MemoryDecodeCache, routing: DecodeRouting) -> torch.Tensor:
    """q (B, [L,] H, 64) over an 8-bit cache (moc_cache8_attend).  The matrix products take bfloat16 queries: others are
    rounded to them, 2^-8 of a query, a sixteenth of the cache's own rounding."""
    q = _aligned(q if q.dtype == torch.bfloat16 else q.to(torch.bfloat16))
    pl, dev = routing.plan, q.device
    out = torch.empty_like(q)
    nbytes = _attend8_workspace(B, Lq, H, cache.HK, routing.NS)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    args = _pack_cache8(q.data_ptr(), cache.k_tiles.data_ptr(), cache.v_tiles.data_ptr(), cache.k_scale.data_ptr(),
                        cache.v_scale.data_ptr(), routing.omega.data_ptr(), routing.idx.data_ptr(), pl.uniq.data_ptr(),
                        pl.n_uniq.data_ptr(), pl.csr_off.data_ptr(), pl.csr_edge.data_ptr(), pl.edge_u.data_ptr(),
                        routing.row_tab.data_ptr(), out.data_ptr(), routing.max_units, B, Lq, pl.num_chapters, H, cache.HK,
                        routing.NS, 0.125)
    with L.on_device(dev):
        call("moc_cache8_attend", args, ws.data_ptr(), nbytes, stream_ptr(dev))
    return out


def _attend_tokens(q: torch.Tensor, cache: MemoryDecodeCache, routing: DecodeRouting) -> torch.Tensor:
    """q (B, L, H, 64) over a float32 or bfloat16 cache: the sequence attention on the cache's tiles."""
    B, Lq, H, D = q.shape
    if cache.T != 64:
        raise ValueError(f"the decode cache's attention needs 64 tokens per chapter, got {cache.T}")
    q = _aligned(q.to(cache.dtype))
    dev, HK = q.device, cache.HK
    idx = torch.where(routing.idx < routing.plan.num_chapters, routing.idx, -1)
    lse = torch.empty(B, H, (Lq + 127) // 128 * 128, device=dev, dtype=torch.float32)
    out = torch.empty_like(q)
    with L.on_device(dev):
        call("moc_xattn_fwd", L.dtype_code(cache.dtype), ptr(q), ptr(cache.k_tiles), ptr(cache.v_tiles), cache.k_tiles.numel(),
             HK * 4096, 4096, 64, ptr(idx), ptr(routing.omega), B, Lq, H, HK, D, 64, routing.NS, 0.125, ptr(out), ptr(lse),
             stream_ptr(dev))
    return out


def decode_attention(q: torch.Tensor, cache: MemoryDecodeCache, routing: DecodeRouting) -> torch.Tensor:
    """q (B, H, 64) -> attention output (B, H, 64) over the routed chapters (joint softmax, omega-weighted), or for
    several query tokens of each sequence (B, L, H, 64) -> (B, L, H, 64), over a float32 or bfloat16 cache of up to 4 GiB
    for K.  The result has the cache's type, bfloat16 over an 8-bit cache."""
    L.require_same_gpu(q, cache.k_tiles, routing.idx)
    if q.dim() not in (3, 4) or q.shape[-1] != 64 or q.shape[0] != routing.B or q.shape[-2] % cache.HK != 0:
        raise ValueError(f"queries of shape {tuple(q.shape)}: expected ({routing.B}, [tokens,] heads, 64) with heads a "
                         f"multiple of {cache.HK}")
    if routing.plan.num_chapters > cache.num_chapters:
        raise ValueError(f"routing over {routing.plan.num_chapters} chapters, cache of {cache.num_chapters}")
    Lq = q.shape[1] if q.dim() == 4 else 1
    if q.numel() == 0 or routing.NS == 0:
        return torch.zeros(q.shape, device=q.device, dtype=torch.bfloat16 if cache.dtype == FP8 else cache.dtype)
    if cache.dtype == FP8:
        return _attend8(q, q.shape[0], Lq, q.shape[-2], cache, routing)
    if q.dim() == 4:
        return _attend_tokens(q, cache, routing)
    B, H, D = q.shape
    if q.dtype != cache.dtype:
        q = q.to(cache.dtype)
    q = q.contiguous()
    dt = L.dtype_code(cache.dtype)
    st = stream_ptr(q.device)
    NS = routing.NS
    E = B * NS
    o_part = torch.empty(E * H, D, device=q.device, dtype=cache.dtype)
    lse_part = torch.empty(E * H, device=q.device, dtype=torch.float32)
    pl = routing.plan
    call("moc_decode_partial", dt, ptr(q), B, H, ptr(cache.k_tiles), ptr(cache.v_tiles), cache.HK, D, cache.T,
         ptr(pl.uniq), ptr(pl.n_uniq), ptr(pl.csr_off), ptr(pl.csr_edge), routing.max_units, ptr(routing.omega), NS,
         float(D) ** -0.5, ptr(o_part), ptr(lse_part), ptr(routing.row_tab), st)
    out = torch.empty(B, H, D, device=q.device, dtype=cache.dtype)
    lse = torch.empty(B * H, device=q.device, dtype=torch.float32)
    call("moc_sparse_combine", dt, ptr(o_part), ptr(lse_part), ptr(pl.edge_u), None, 1, NS, H, B, H, 0, ptr(out),
         ptr(lse), st)
    return out


class PagedKVCache:
    """Keys and values of several sequences in pages of a pool, for tokens that attend to what came before them (or to
    an encoder's states).  Inference only.

    ``k_pages``, ``v_pages`` (pages, page size, kv heads, 64 or 128), float32 or bfloat16, the page size a multiple of 16;
    they may be views with strides of their own (16-byte pieces).  ``block_table`` (sequences, pages of one) int32: token t
    of sequence b lies in row t % page size of page block_table[b, t // page size]; entries outside the pool hold nothing:
    what is written there is dropped, and keys there do not count.  ``lengths`` (sequences,) int32: tokens held.  The
    server owns all four tensors and writes table and lengths as it hands out pages (in place: another tensor needs another
    PagedKVCache); the kernels read them on the device, so a captured step stays right when they change."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError(f"pages of shapes {tuple(k_pages.shape)}, {tuple(v_pages.shape)}: expected two equal (pages, page "
                             "size, kv heads, head dim)")
        if k_pages.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"pages must be float32 or bfloat16, got {k_pages.dtype}")
        if k_pages.shape[1] == 0 or k_pages.shape[1] % 16 or k_pages.shape[2] == 0 or k_pages.shape[3] not in (64, 128):
            raise ValueError(f"pages of {k_pages.shape[1]} tokens, {k_pages.shape[2]} kv heads, {k_pages.shape[3]} dims: expected "
                             "a multiple of 16 tokens, heads of 64 or 128")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1:
            raise ValueError("block_table must be (sequences, pages) int32 with its rows in one piece")
        if lengths.shape != block_table.shape[:1] or lengths.dtype != torch.int32 or not lengths.is_contiguous():
            raise ValueError(f"lengths must be ({block_table.shape[0]},) int32, contiguous")
        L.require_same_gpu(k_pages, v_pages, block_table, lengths)
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            es = t.element_size()
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(s * es % 16 for s in t.stride()[:3]):
                raise ValueError(f"{name} must be rows in 16-byte pieces")
            if t.stride(1) < t.shape[3] or t.stride(1) * es >= 1 << 24:
                raise ValueError(f"{name}: rows that overlap, or lie 16 MiB or more apart")
        self.k_pages, self.v_pages, self.block_table, self.lengths = k_pages, v_pages, block_table, lengths
        # what every call hands to the kernels of them, worked out once (a step is two launches: its host time counts)
        P, page, HK, D = k_pages.shape
        self._sizes = (P, page, HK, D, block_table.shape[0], block_table.shape[1])
        self._k_strides, self._v_strides = k_pages.stride()[:3], v_pages.stride()[:3]
        self._table = (block_table.stride(0), P, block_table.shape[1], page)
        self._code = L.dtype_code(k_pages.dtype)

    def __setattr__(self, name, value):
        if name in ("k_pages", "v_pages", "block_table", "lengths") and name in self.__dict__ and value is not self.__dict__[name]:
            raise AttributeError(f"{name} is written to in place: its checks and strides are those of the cache's construction")
        super().__setattr__(name, value)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, sequences: int, max_pages: int, *,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> "PagedKVCache":
        """An empty cache: no sequence holds a page (table entries -1) or a token."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        shape = (num_pages, page_size, num_kv_heads, head_dim)
        return cls(torch.zeros(shape, device=dev, dtype=dtype), torch.zeros(shape, device=dev, dtype=dtype),
                   torch.full((sequences, max_pages), -1, device=dev, dtype=torch.int32),
                   torch.zeros(sequences, device=dev, dtype=torch.int32))

    @classmethod
    @torch.no_grad()
    def from_memory(cls, memory_attn, memory: torch.Tensor, memory_lengths: Optional[torch.Tensor] = None, *,
                    page_size: int = 64, memory_positions: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """The keys and values of MemoryCrossAttention over an encoder's states (B, N, d), projected once for a
        generation (``memory_decode_step``); pages lie in the order of the sequences.  ``memory_lengths`` (B,) as in its
        forward; ``memory_positions`` as there.  A float16 module's pages are float32, as its attention is."""
        if memory.dim() != 3 or memory.shape[0] * memory.shape[1] == 0:
            raise ValueError(f"memory must be (B, N, d) with states, got {tuple(memory.shape)}")
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"pages of {page_size} tokens: expected a multiple of 16")
        B, N, _ = memory.shape
        k, v = memory_attn.project_memory(memory, memory_positions)
        per = (N + page_size - 1) // page_size
        dtype = k.dtype if k.dtype in (torch.float32, torch.bfloat16) else torch.float32
        self = cls.allocate(B * per, page_size, k.shape[2], k.shape[3], B, per, dtype=dtype, device=k.device)
        self.block_table.copy_(torch.arange(B * per, device=k.device, dtype=torch.int32).view(B, per))
        self.append(k, v)
        if memory_lengths is not None:
            if tuple(memory_lengths.shape) != (B,) or memory_lengths.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"memory_lengths of shape {tuple(memory_lengths.shape)}, expected ({B},) int32 or int64")
            self.lengths.copy_(memory_lengths.clamp(0, N))
        return self

    @property
    def page_size(self) -> int:
        return self.k_pages.shape[1]

    @property
    def dtype(self) -> torch.dtype:
        return self.k_pages.dtype

    def append(self, k: torch.Tensor, v: torch.Tensor, *, positions: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, norm: Optional[bool] = None,
               inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
        """Writes new tokens' keys and values, k and v (sequences, tokens, kv heads, head dim), behind what the sequences
        hold, and adds them to ``lengths``.  With ``positions`` (sequences,), int32 or int64, token i of sequence b goes to
        place positions[b] + i instead and ``lengths`` stays the server's.  A token whose place has no page is dropped.

        Keys may be normed and rotated on the way (``k_weight``, ``norm``, ``inv_freq``, ``interleaved`` as in
        ``ops.qk_norm_rotate``, ``norm`` where a weight is given by default; the position is the token's place), and the
        queries ``q`` of the same tokens with them: returns q so treated.  One launch.  k, v and q of another type than
        the cache's are rounded to it first."""
        _, _, HK, D, B, _ = self._sizes
        shape = k.shape
        if len(shape) != 4 or shape != v.shape or shape[0] != B or shape[2] != HK or shape[3] != D:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)}: expected ({B}, tokens, {HK}, {D})")
        T = shape[1]
        if q is not None and (q.dim() != 4 or q.shape[0] != B or q.shape[1] != T or q.shape[3] != D or q.shape[2] == 0):
            raise ValueError(f"q {tuple(q.shape)}: expected ({B}, {T}, heads, {D})")
        if positions is not None and (tuple(positions.shape) != (B,) or positions.dtype not in (torch.int32, torch.int64)):
            raise ValueError(f"positions of shape {tuple(positions.shape)} {positions.dtype}, expected ({B},) int32 or int64")
        weighed = q_weight is not None or k_weight is not None
        if norm is None:
            norm = weighed
        if weighed and not norm:
            raise ValueError("a weight needs norm=True")
        if q is None and q_weight is not None:
            raise ValueError("q_weight without q")
        if not (k.is_floating_point() and v.is_floating_point()) or (q is not None and not q.is_floating_point()):
            raise ValueError("k, v and q must be floating-point")
        L.require_same_gpu(self.k_pages, k, v, q, positions, q_weight, k_weight, inv_freq)
        kw = ops._head_weight(k_weight, HK, D, "k_weight")
        qw = None if q is None else ops._head_weight(q_weight, q.shape[2], D, "q_weight")
        freq = ops._head_frequencies(inv_freq, D)
        place = self.lengths if positions is None else positions
        # (pointer, batch stride, row stride, step) of the places; the page table
        at, pos32 = (place.stride(0), 0, 1), int(place.dtype == torch.int32)
        tb, P, most, page = self._table
        where, table = place.data_ptr(), self.block_table.data_ptr()
        turns = freq is not None
        k, v = self._rows(k), self._rows(v)
        pack = ops._pack_head_rows
        sets = [pack(k.data_ptr(), L.ptr0(kw), self.k_pages.data_ptr(), 0, 0, 0, where, table, *k.stride()[:3], *self._k_strides,
                     *at, tb, B, T, P, most, HK, int(kw is not None and kw.dim() == 2), int(norm), int(turns), pos32, page),
                pack(v.data_ptr(), 0, self.v_pages.data_ptr(), 0, 0, 0, where, table, *v.stride()[:3], *self._v_strides, *at, tb,
                     B, T, P, most, HK, 0, 0, 0, pos32, page)]
        out = None
        if q is not None:
            q = self._rows(q)
            H = q.shape[2]
            out = torch.empty(B, T, H, D, device=q.device, dtype=q.dtype)
            sets.append(pack(q.data_ptr(), L.ptr0(qw), out.data_ptr(), 0, 0, 0, where, 0, *q.stride()[:3], T * H * D, H * D, D, *at,
                             0, B, T, 0, 0, H, int(qw is not None and qw.dim() == 2), int(norm), int(turns), pos32, 0))
        dev = k.device
        with L.on_device(dev):
            call("moc_head_rotate_fwd", ops._head_args(sets, freq, D, interleaved, self.dtype, float(eps)), stream_ptr(dev))
            if positions is None:
                self.lengths.add_(T)
        return out

    def _rows(self, x: torch.Tensor) -> torch.Tensor:
        x = x.detach()
        if x.dtype != self.k_pages.dtype:
            x = x.to(self.k_pages.dtype)
        return x if x.stride(3) == 1 else x.contiguous()


def paged_attention(q: torch.Tensor, cache: PagedKVCache, *, causal: bool = False,
                    softmax_scale: Optional[float] = None) -> torch.Tensor:
    """Attention of new tokens over their sequences' pages: q (B, H, D) or several tokens (B, L, H, D) -> the same shape
    in the cache's type.  Each sees the ``cache.lengths`` first keys of its sequence; with ``causal`` token l of L the
    first lengths - L + l + 1 (the tokens are the last ones appended; the values of the newer ones, which it gives no
    weight, must be finite all the same).  Of those, keys past the table's end or in no page do not exist (appended, they
    were dropped), and what lies there or behind a sequence's length may be anything.  A token that sees no key gets 0."""
    P, page, HK, D, B, most = cache._sizes
    shape = q.shape
    if len(shape) not in (3, 4) or shape[0] != B or shape[-1] != D or shape[-2] == 0 or shape[-2] % HK:
        raise ValueError(f"queries of shape {tuple(q.shape)}: expected ({B}, [tokens,] heads, {D}) with heads a multiple of {HK}")
    scale = float(D) ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < 2.0 ** 127:
        raise ValueError(f"softmax_scale must be positive and less than 2^127, got {softmax_scale}")
    if not q.is_floating_point():
        raise ValueError(f"queries of {q.dtype}")
    L.require_same_gpu(cache.k_pages, q)
    q = q.detach()
    x = q.unsqueeze(1) if len(shape) == 3 else q
    x = ops._attn_rows(x if x.dtype == cache.dtype else x.to(cache.dtype), False)
    Lq, H = x.shape[1], x.shape[2]
    if B == 0 or Lq == 0 or most == 0 or P == 0:
        return torch.zeros(shape, device=q.device, dtype=cache.dtype)
    dev = q.device
    out = torch.empty(shape, device=dev, dtype=cache.dtype)
    nbytes = ops.kv_decode_workspace(B, Lq, most * page, H, HK, D, cache._code)
    (kp, kn, kh), (vp, vn, vh) = cache._k_strides, cache._v_strides
    args = ops.pack_kv_decode(x.data_ptr(), cache.k_pages.data_ptr(), cache.v_pages.data_ptr(), out.data_ptr(),
                              cache.lengths.data_ptr(), cache.block_table.data_ptr(), 0, *ops._strides3(x), 0, kn, kh, 0, vn, vh,
                              kp, vp, cache._table[0], B, Lq, 0, P, most, H, HK, D, cache._code, page, int(causal), scale)
    with L.on_device(dev):
        if nbytes:
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            call("moc_kv_decode", args, ws.data_ptr(), nbytes, stream_ptr(dev))
        else:
            call("moc_kv_decode", args, None, 0, stream_ptr(dev))
    return out


def _step_native(x, wq, wo, H: int, cache: MemoryDecodeCache, routing: DecodeRouting) -> bool:
    """Whether moc_decode_step takes the step (bf16 throughout, few rows; with the per-kernel timing armed
    the kernels run as separate entry points).  A re-routed step of 16 sequences: 172 to 182 us with a call
    per kernel, most of it host time, 91 with three calls."""
    return (cache.dtype == torch.bfloat16 and wo.dtype == torch.bfloat16 and 0 < x.shape[0] == routing.B
            and ops._few_rows(x, wq) and wo.is_cuda and H % 2 == 0 and wq.shape == (64 * H, x.shape[1])
            and wo.shape[0] % 16 == 0 and wo.shape[1] == 64 * H and cache.k_tiles.is_cuda and H % cache.HK == 0
            and x.data_ptr() % 16 == 0 and wq.data_ptr() % 16 == 0 and wo.data_ptr() % 16 == 0
            and L.KERNEL_EVENTS is None)


def _states_step(memory_attn, hidden: torch.Tensor, cache: PagedKVCache, positions) -> torch.Tensor:
    """memory_decode_step over an encoder's states."""
    B, Lx = hidden.shape[0], hidden.shape[1] if hidden.dim() == 3 else 1
    H, D = memory_attn.num_heads, memory_attn.head_dim
    wq, wo = memory_attn.q_proj.weight, memory_attn.o_proj.weight
    if (positions is not None) != (memory_attn.rotary_dim > 0):
        raise ValueError("positions are given for a module that rotates its heads (rotary_dim), and only then")
    if hidden.numel() == 0:
        return torch.zeros(B, Lx, wo.shape[0], device=hidden.device, dtype=wo.dtype)
    q = ops.linear(hidden.reshape(B, Lx, -1).to(wq.dtype), wq).view(B, Lx, H, D)
    q = memory_attn.treat_queries(q, positions)
    a = paged_attention(q, cache, softmax_scale=memory_attn.scale)
    return ops.linear(a.reshape(B, Lx, H * D).to(wo.dtype), wo)


def memory_decode_step(memory_attn, hidden: torch.Tensor, cache, routing: Optional[DecodeRouting] = None, *,
                       positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step of a memory sublayer: hidden (B, 1, d) -> (B, 1, d) (before the residual); or L tokens
    of each sequence, (B, L, d) -> (B, L, d), over one routing (a prompt served from the cache).

    Over an encoder's states: ``cache`` is a PagedKVCache (``PagedKVCache.from_memory``), there is no routing, and a
    module that rotates its heads needs the tokens' ``positions``, (L,) or (B, L)."""
    B = hidden.shape[0]
    H = memory_attn.num_heads
    if isinstance(cache, PagedKVCache):
        if routing is not None:
            raise ValueError("a PagedKVCache takes no routing")
        with torch.no_grad():
            return _states_step(memory_attn, hidden, cache, positions)
    if routing is None:
        raise ValueError("a MemoryDecodeCache needs its routing")
    if positions is not None or getattr(memory_attn, "treats_heads", False):
        raise ValueError("positions, qk_norm and rotary_dim are for an encoder's states (PagedKVCache)")
    with torch.no_grad():
        wq, wo = memory_attn.q_proj.weight, memory_attn.o_proj.weight
        if hidden.dim() == 3 and hidden.shape[1] != 1:
            Lx = hidden.shape[1]
            if hidden.numel() == 0:
                return torch.zeros(B, Lx, wo.shape[0], device=hidden.device, dtype=wo.dtype)
            q = ops.linear(hidden.to(wq.dtype), wq).view(B, Lx, H, memory_attn.head_dim)
            a = decode_attention(q, cache, routing)
            return ops.linear(a.reshape(B, Lx, H * memory_attn.head_dim).to(wo.dtype), wo)
        x = hidden.reshape(B, -1).to(wq.dtype)
        if _step_native(x, wq, wo, H, cache, routing):
            x, wq, wo = x.contiguous(), wq.contiguous(), wo.contiguous()
            pl, NS, N = routing.plan, routing.NS, wo.shape[0]
            nbytes = L.query("moc_decode_step_workspace", B, H, NS)
            ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
            out = torch.empty(B, 1, N, device=x.device, dtype=x.dtype)
            call("moc_decode_step", ptr(x), B, x.shape[1], ptr(wq), H, ptr(cache.k_tiles), ptr(cache.v_tiles), cache.HK,
                 cache.T, ptr(pl.uniq), ptr(pl.n_uniq), ptr(pl.csr_off), ptr(pl.csr_edge), ptr(pl.edge_u),
                 routing.max_units, ptr(routing.omega), NS, 0.125, ptr(wo), N, ptr(ws), nbytes, ptr(out),
                 ptr(routing.row_tab), stream_ptr(x.device))
            return out
        q = ops.linear(x, wq).view(B, H, memory_attn.head_dim)
        a = decode_attention(q, cache, routing)
        return ops.linear(a.reshape(B, 1, -1).to(wo.dtype), wo)


class _Layer(ctypes.Structure):
    """moc_decode_layer."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "wq", "k_tiles", "v_tiles", "wo", "uniq", "n_uniq", "csr_off",
                                               "csr_edge", "edge_u", "row_tab", "omega", "workspace", "out")]
    _fields_.append(("max_u", ctypes.c_int64))


def _group_native(layers, inputs) -> bool:
    """Whether the layers' steps run as one group (moc_decode_step_group): several, each on the one-call
    step, of one shape, with the slot counts its combine kernel takes."""
    shapes = set()
    for (attn, cache, routing), h in zip(layers, inputs):
        if isinstance(cache, PagedKVCache) or getattr(attn, "treats_heads", False):
            return False
        wq, wo, H = attn.q_proj.weight, attn.o_proj.weight, attn.num_heads
        if h.dtype != wq.dtype or not (h.is_contiguous() and wq.is_contiguous() and wo.is_contiguous()):
            return False
        x = h.reshape(h.shape[0], -1)
        if not _step_native(x, wq, wo, H, cache, routing) or cache.T != 64 or x.device != inputs[0].device:
            return False
        shapes.add((x.shape, H, cache.HK, routing.NS, wo.shape))
    return len(layers) > 1 and len(shapes) == 1 and 8 < routing.NS <= 68 and routing.B * H <= 16384


def _decode_steps(layers, inputs):
    """memory_decode_step of every layer of a group, one launch per kernel for all of them."""
    with torch.no_grad():
        x = inputs[0]
        B, dev = x.shape[0], x.device
        attn, cache, routing = layers[0]
        H, NS, N = attn.num_heads, routing.NS, attn.o_proj.weight.shape[0]
        nbytes = L.query("moc_decode_step_workspace", B, H, NS)
        ws = torch.empty(len(layers), nbytes, device=dev, dtype=torch.uint8)
        outs = [torch.empty(B, 1, N, device=dev, dtype=x.dtype) for _ in layers]
        args = (_Layer * len(layers))()
        for i, ((attn, c, r), h) in enumerate(zip(layers, inputs)):
            p = r.plan
            args[i] = _Layer(ptr(h), ptr(attn.q_proj.weight), ptr(c.k_tiles), ptr(c.v_tiles), ptr(attn.o_proj.weight),
                             ptr(p.uniq), ptr(p.n_uniq), ptr(p.csr_off), ptr(p.csr_edge), ptr(p.edge_u), ptr(r.row_tab),
                             ptr(r.omega), ws[i].data_ptr(), ptr(outs[i]), r.max_units)
        call("moc_decode_step_group", ctypes.addressof(args), len(layers), B, x.numel() // B, H, cache.HK, cache.T, NS,
             0.125, N, nbytes, stream_ptr(dev))
        return outs


class DecodeStepGraph:
    """The per-token decode of several memory sublayers captured once as a HIP graph
    (torch.cuda.CUDAGraph) and replayed for every generated token: one graph launch replaces
    the ~4 kernel launches per layer, and their inter-launch gaps.  Layers of one shape are captured
    together, one launch per kernel for all of them (every layer's input is given at once).

    ``layers`` is a list of (memory_attn, cache, routing); ``inputs`` the per-layer hidden
    states (B, 1, d) used for the capture (their shapes and dtypes are fixed).  ``run(inputs)``
    copies new hidden states into the captured input buffers, replays, and returns the
    per-layer outputs (buffers owned by the graph, overwritten by the next replay).  The
    routing and the caches must stay alive and unchanged while the graph is used."""

    def __init__(self, layers, inputs, warmup: int = 2):
        if len(layers) != len(inputs):
            raise ValueError("one input per layer")
        self.layers = list(layers)
        self.static_in = [x.detach().clone() for x in inputs]
        stream = torch.cuda.Stream(device=self.static_in[0].device)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(warmup):
                self._body()
        torch.cuda.current_stream().wait_stream(stream)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.static_out = self._body()

    def _body(self):
        if _group_native(self.layers, self.static_in):
            return _decode_steps(self.layers, self.static_in)
        return [memory_decode_step(attn, x, cache, routing)
                for (attn, cache, routing), x in zip(self.layers, self.static_in)]

    def run(self, inputs):
        """Replay with ``inputs`` (copied into the captured input buffers unless they are those
        buffers: a serving loop that writes each token's hidden states into ``static_in``
        directly replays with no copies)."""
        new = [(buf, x) for buf, x in zip(self.static_in, inputs) if x.data_ptr() != buf.data_ptr()]
        if len(new) > 1 and all(x.shape == buf.shape and x.dtype == buf.dtype and x.device == buf.device for buf, x in new):
            torch._foreach_copy_([buf for buf, _ in new], [x for _, x in new])
        else:
            for buf, x in new:
                buf.copy_(x)
        self.graph.replay()
        return self.static_out
