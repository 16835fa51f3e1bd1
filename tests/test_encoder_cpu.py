"""Refusals of the encoder attention, the head norms and the paged cache that need no GPU: shapes, types, options."""

import ctypes

import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("q,k,kw,match", [
    ((2, 3, 4, 64), (2, 5, 3, 64), {}, "query heads"),
    ((2, 3, 4, 80), (2, 5, 2, 80), {}, "64 or 128"),
    ((2, 3, 4, 64), (2, 5, 2, 128), {}, "expected"),
    ((2, 3, 4, 64), (3, 5, 2, 64), {}, "expected"),
    ((2, 3, 64), (2, 5, 64), {}, "expected"),
    ((2, 3, 4, 64), (2, 5, 2, 64), dict(softmax_scale=0.0), "softmax_scale"),
    ((2, 3, 4, 64), (2, 5, 2, 64), dict(softmax_scale=float("nan")), "softmax_scale"),
    ((2, 3, 4, 64), (2, 5, 2, 64), dict(softmax_scale=-1.0), "softmax_scale"),
])
def test_cross_attention_shapes(q, k, kw, match):
    from memory_amd import ops
    with pytest.raises(ValueError, match=match):
        ops.cross_attention(rnd(*q), rnd(*k), rnd(*k), **kw)


def test_cross_attention_types_and_device():
    from memory_amd import ops
    q, k = rnd(2, 3, 4, 64), rnd(2, 5, 2, 64)
    with pytest.raises(ValueError, match="one floating-point type"):
        ops.cross_attention(q, k.bfloat16(), k.bfloat16())
    with pytest.raises(ValueError, match="one floating-point type"):
        ops.cross_attention(q.int(), k.int(), k.int())
    with pytest.raises(ValueError, match="expected"):
        ops.cross_attention(q, k, k[:, :4])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cross_attention(q, k, k)


@pytest.mark.parametrize("x,w,kw,match", [
    ((2, 3, 4, 63), None, {}, "head dim even"),
    ((2, 3, 4, 514), None, {}, "head dim even"),
    ((2, 3, 64), None, {}, "expected"),
    ((2, 3, 4, 64), (4,), dict(norm=False), "norm=True"),
    ((2, 3, 4, 64), None, dict(norm=False), "nothing to do"),
    ((2, 3, 4, 64), None, dict(positions=torch.arange(3)), "inv_freq"),
])
def test_head_rotate_arguments(x, w, kw, match):
    from memory_amd import ops
    with pytest.raises(ValueError, match=match):
        ops.head_norm_rotate(rnd(*x), None if w is None else rnd(*w), **kw)


def test_head_rotate_pairs_and_device():
    from memory_amd import ops
    with pytest.raises(ValueError, match="one head dim"):
        ops.qk_norm_rotate(rnd(1, 2, 4, 64), rnd(1, 2, 4, 32))
    with pytest.raises(ValueError, match="one head dim"):
        ops.qk_norm_rotate(rnd(1, 2, 4, 64), rnd(1, 2, 4, 64, dtype=BF))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.head_norm_rotate(rnd(1, 2, 4, 64))
    for bad in ((3, 10000.0), (0, 10000.0), (-2, 10000.0), (64, 0.0), (64, float("nan"))):
        with pytest.raises(ValueError):
            ops.rope_frequencies(*bad)
    f = ops.rope_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0 and abs(f[16].item() - 1e-2) < 1e-15


@pytest.mark.parametrize("k,v,table,lens,match", [
    (rnd(4, 16, 2, 64), rnd(4, 16, 2, 128), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "equal"),
    (rnd(4, 16, 2, 64), rnd(4, 16, 2, 64, dtype=BF), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "equal"),
    (rnd(4, 16, 2, 64).half(), rnd(4, 16, 2, 64).half(), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "float32 or"),
    (rnd(4, 24, 2, 64), rnd(4, 24, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "multiple of 16"),
    (rnd(4, 16, 2, 96), rnd(4, 16, 2, 96), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "64 or 128"),
    (rnd(4, 16, 2, 64), rnd(4, 16, 2, 64), torch.zeros(2, 2), torch.zeros(2, dtype=torch.int32), "block_table"),
    (rnd(4, 16, 2, 64), rnd(4, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), "lengths"),
    (rnd(4, 16, 2, 64), rnd(4, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2), "lengths"),
])
def test_paged_cache_tensors(k, v, table, lens, match):
    from memory_amd.decode import PagedKVCache
    with pytest.raises(ValueError, match=match):
        PagedKVCache(k, v, table, lens)


def test_paged_cache_device():
    from memory_amd.decode import PagedKVCache
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagedKVCache(rnd(4, 16, 2, 64), rnd(4, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_paged_cache_tensors_stay():
    """Another tensor of another shape or type would be read with the strides of the first."""
    from memory_amd.decode import PagedKVCache
    cache = PagedKVCache.__new__(PagedKVCache)
    for name in ("k_pages", "v_pages", "block_table", "lengths"):
        t = torch.zeros(4, dtype=torch.int32)
        setattr(cache, name, t)
        with pytest.raises(AttributeError, match="in place"):
            setattr(cache, name, torch.zeros(2, dtype=torch.int64))
        cache.__dict__[name].add_(1)
        setattr(cache, name, getattr(cache, name))     # (what `cache.lengths += 1` does)
        assert getattr(cache, name) is t
    cache.owner = 1


def test_module_options():
    from memory_amd.memory_attention import MemoryCrossAttention
    for kw in (dict(rotary_dim=63), dict(rotary_dim=128), dict(rotary_dim=-2), dict(rotary_dim=64, rotary_base=0.0)):
        with pytest.raises(ValueError):
            MemoryCrossAttention(256, 4, **kw)
    m = MemoryCrossAttention(256, 4, 2, qk_norm=True)
    assert {n for n, _ in m.named_parameters()} >= {"q_norm.weight", "k_norm.weight"}
    assert not any("norm" in n for n, _ in MemoryCrossAttention(256, 4, 2).named_parameters())
    h, mem = rnd(1, 3, 256), rnd(1, 64, 256)
    routed = dict(bank=rnd(64, 256), chapter_indices=torch.zeros(1, 1), chapter_weights=rnd(1, 1), num_chapters=1, tokens_per_chapter=64)
    with pytest.raises(ValueError, match="dense memory"):
        m(h, routed_memory_state=routed)
    with pytest.raises(ValueError, match="dense memory"):
        MemoryCrossAttention(256, 4, 2)(h, routed_memory_state=routed, memory_lengths=torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="rotary_dim"):
        m(h, mem, query_positions=torch.arange(3))
    with pytest.raises(ValueError, match="return_attn_weights"):
        m(h, mem, memory_mask=torch.ones(1, 64, dtype=torch.bool), return_attn_weights=True)


def test_entry_points_refuse():
    """Nothing is launched: the library's own checks of what it is given."""
    from memory_amd import _lib as L
    from memory_amd import ops

    def cross(name, *, q=16, dtype=L.MOC_BF16, D=64, H=4, HK=2, B=1, Lq=3, N=5, kn=128, scale=0.125, ws=None, qb=0, lse=16, dk=16,
              dv=16):
        a = ops._pack_cross(q, 16, 16, 16, 16, 0, 16, dk, dv, lse, 0, 0, qb, 256, 64, 0, kn, 64, 0, kn, 64, 0, 256, 64, B, Lq, N,
                            H, HK, D, dtype, scale)
        L.call(name, a, ws, 0, None)

    for kw, match in ((dict(dtype=7), "dtype"), (dict(D=96), "head dim"), (dict(H=5), "heads"), (dict(HK=0), "heads"),
                      (dict(N=0), "empty"), (dict(B=0), "empty"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
                      (dict(q=8), "aligned"), (dict(kn=67), "strides"), (dict(kn=32), "overlap"), (dict(kn=1 << 24), "16 MiB"),
                      (dict(qb=-8), "strides"), (dict(q=0), "null"), (dict(N=1 << 30), "sizes")):
        with pytest.raises(ValueError, match=match):
            cross("moc_cross_fwd", **kw)
    for kw, match in ((dict(lse=0), "null"), (dict(dk=0), "together"), (dict(), "workspace")):
        with pytest.raises(ValueError, match=match):
            cross("moc_cross_bwd", **kw)
    with pytest.raises(ValueError, match="workspace"):
        cross("moc_cross_fwd", N=4096)

    def decode(*, table=16, lengths=16, page=16, words=0, num_pages=4):
        a = ops.pack_kv_decode(16, 16, 16, 16, lengths, table, words, 0, 256, 64, 0, 128, 64, 0, 128, 64, 2048, 2048, 4, 1, 1, 0,
                               num_pages, 4, 4, 2, 64, L.MOC_BF16, page, 0, 0.125)
        L.call("moc_kv_decode", a, None, 0, None)

    for kw, match in ((dict(lengths=0), "lengths"), (dict(words=16), "mask"), (dict(page=24), "multiple of 16"),
                      (dict(page=0), "empty"), (dict(num_pages=-1), "table")):
        with pytest.raises(ValueError, match=match):
            decode(**kw)

    def heads(*, D=64, R=64, dtype=L.MOC_BF16, freq=16, H=4, x=16, w=0, norm=1, B=1, Lq=2, nseg=1):
        f = ops._pack_head_rows(x, w, 16, 16, 16, 0, 0, 0, 0, 256, 64, 0, 256, 64, 0, 0, 1, 0, B, Lq, 0, 0, H, 0, norm, 1, 0, 0)
        a = f * nseg + ops._NO_ROWS * (3 - nseg) + ops._pack_head_tail(freq, nseg, D, R, 0, dtype, 1e-6)
        L.call("moc_head_rotate_fwd", a, None)

    for kw, match in ((dict(D=63), "head dim"), (dict(D=514), "head dim"), (dict(R=66), "rotated"), (dict(R=3), "rotated"),
                      (dict(dtype=5), "dtype"), (dict(freq=0), "frequencies"), (dict(H=0), "sizes"), (dict(x=0), "null"),
                      (dict(w=16, norm=0), "weight"), (dict(B=1 << 16, Lq=1 << 16), "tokens")):
        with pytest.raises(ValueError, match=match):
            heads(**kw)
    assert ctypes.sizeof(ops._HeadRows) == 200


def test_decode_step_arguments():
    """A cache of pages takes no routing, a module that rotates needs positions, another takes none; a routed layer
    refuses an attention module that norms or rotates its heads."""
    from memory_amd.decode import PagedKVCache, _group_native, memory_decode_step
    from memory_amd.memory_attention import MemoryCrossAttention
    from memory_amd.model import RoutedMemoryLayer
    cache = PagedKVCache.__new__(PagedKVCache)
    plain, turning = MemoryCrossAttention(256, 4, 2), MemoryCrossAttention(256, 4, 2, rotary_dim=64)
    h = rnd(2, 1, 256)
    with pytest.raises(ValueError, match="no routing"):
        memory_decode_step(plain, h, cache, object())
    with pytest.raises(ValueError, match="positions are given"):
        memory_decode_step(plain, h, cache, positions=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="positions are given"):
        memory_decode_step(turning, h, cache)
    with pytest.raises(ValueError, match="needs its routing"):
        memory_decode_step(plain, h, object())
    with pytest.raises(ValueError, match="PagedKVCache"):
        memory_decode_step(turning, h, object(), object())
    assert not _group_native([(plain, cache, None)] * 2, [h, h])
    layer = RoutedMemoryLayer(256, 4, num_chapters=4, tokens_per_chapter=64, top_k=2)
    layer.memory_attn = MemoryCrossAttention(256, 4, qk_norm=True)
    assert layer._fused(h, rnd(256, 256)) is None


def test_pages_without_a_table():
    """Rows of pages never become rows in a piece: a page size without a table is taken only where the table has no
    columns (whose tensor has no address), and a table without a page size is refused."""
    from memory_amd import _lib as L
    from memory_amd import ops
    assert torch.empty(2, 0, dtype=torch.int32).data_ptr() == 0

    def heads(*, y=16, table=16, page=16, pages=4, most=3, B=1, name="moc_head_rotate_fwd"):
        f = ops._pack_head_rows(16, 0, y, 16, 16, 0, 16, table, 256, 64, 64, 2048, 128, 64, 0, 0, 1, most, B, 2, pages, most, 2, 0,
                                1, 0, 0, page)
        a = f + ops._NO_ROWS * 2 + ops._pack_head_tail(0, 1, 64, 0, 0, L.MOC_BF16, 1e-6)
        L.call(name, a, *(() if name.endswith("fwd") else (None, 0)), None)

    for kw in (dict(table=0), dict(table=0, pages=0), dict(page=0), dict(page=-16), dict(most=-1), dict(pages=-1),
               dict(name="moc_head_rotate_bwd")):
        with pytest.raises(ValueError, match="pages"):
            heads(**kw)
    for kw in (dict(y=0), dict(y=0, page=0, table=0)):
        with pytest.raises(ValueError, match="null"):
            heads(**kw)
    heads(B=0, table=0)     # (no sequences: nothing is launched)


@pytest.mark.parametrize("scale", [2.0 ** 127, 2.5e38])
def test_scales_that_overflow_in_base_two(scale):
    """scale log2(e) past float32 would make NaN of logits of 0."""
    from memory_amd import _lib as L
    from memory_amd import ops
    from memory_amd.decode import PagedKVCache, paged_attention
    with pytest.raises(ValueError, match="softmax_scale"):
        ops.cross_attention(rnd(2, 3, 4, 64), rnd(2, 5, 2, 64), rnd(2, 5, 2, 64), softmax_scale=scale)
    cache = PagedKVCache.__new__(PagedKVCache)
    cache._sizes = (4, 16, 2, 64, 2, 2)
    with pytest.raises(ValueError, match="softmax_scale"):
        paged_attention(rnd(2, 4, 64), cache, softmax_scale=scale)
    args = ops._pack_cross(16, 16, 16, 16, 16, 0, 16, 16, 16, 16, 0, 0, 0, 256, 64, 0, 128, 64, 0, 128, 64, 0, 256, 64, 1, 3, 5, 4,
                           2, 64, L.MOC_BF16, scale)
    with pytest.raises(ValueError, match="scale"):
        L.call("moc_cross_fwd", args, None, 0, None)


@pytest.mark.parametrize("page_size", [0, -16, 24])
def test_from_memory_page_size(page_size):
    from memory_amd.decode import PagedKVCache
    from memory_amd.memory_attention import MemoryCrossAttention
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedKVCache.from_memory(MemoryCrossAttention(256, 4, 2), rnd(1, 3, 256), page_size=page_size)
