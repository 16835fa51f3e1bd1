"""PagedKVCache and paged_attention against float64 over the keys and values that the pages stand for.

Tolerances: as in test_gpu_cross_attention.py, with the operands' rounding 2^-16 (bfloat16 probabilities go in two
pieces); written rows as in test_gpu_head_rotate.py."""

import pytest
import torch

from helpers import gen
import test_gpu_cross_attention as ca
import test_gpu_head_rotate as hr

BF, F32 = torch.bfloat16, torch.float32


def pool(dev, dt, lens, page, HK, D, room=0, seed=0, spare=3):
    """A cache filled with N(0, 1), pages in random order, NaN behind every sequence and in the spare pages."""
    from memory_amd.decode import PagedKVCache
    g = gen(seed)
    per = max(1, max((n + room + page - 1) // page for n in lens))
    P = len(lens) * per + spare
    table = torch.randperm(P, generator=g)[:len(lens) * per].view(len(lens), per).int()
    k, v = (torch.full((P, page, HK, D), float("nan")) for _ in range(2))
    dense = []
    for b, n in enumerate(lens):
        kk, vv = torch.randn(n, HK, D, generator=g).to(dt), torch.randn(n, HK, D, generator=g).to(dt)
        for t in range(n):
            k[table[b, t // page], t % page], v[table[b, t // page], t % page] = kk[t].float(), vv[t].float()
        dense.append((kk.to(dev), vv.to(dev)))
    cache = PagedKVCache(k.to(dt).to(dev), v.to(dt).to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev))
    return cache, dense


def expect(q, dense, causal=False, holes=None):
    """(result, bound) of q (B, L, H, D) sequence by sequence and row by row"""
    ref, bound = torch.zeros(q.shape, device=q.device, dtype=torch.float64), torch.zeros(q.shape, device=q.device, dtype=torch.float64)
    B, L, H, D = q.shape
    for b, (k, v) in enumerate(dense):
        n = k.shape[0]
        for l in range(L):
            see = max(0, n - L + l + 1) if causal else n
            live = torch.arange(n, device=q.device) < see
            if holes is not None:
                live = live & ~holes[b][:n]
            if n == 0 or not live.any():
                continue
            # (of one row: few rows of a kv head, so two pieces)
            ref[b, l], bound[b, l] = (x[0, 0] for x in ca.reference(q[b:b + 1, l:l + 1], k[None], v[None], live[None]))
    return ref, bound


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("heads", [(4, 4, 64), (8, 2, 128), (16, 1, 64), (24, 1, 128)])
def test_single_tokens(gpu_device, heads, page, dt):
    from memory_amd.decode import paged_attention
    H, HK, D = heads
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 300]
    cache, dense = pool(gpu_device, dt, lens, page, HK, D)
    q = torch.randn(len(lens), H, D, generator=gen(1)).to(dt).to(gpu_device)
    o = paged_attention(q, cache)
    ref, bound = expect(q[:, None], dense)
    ca.close(o[:, None], ref, bound, "out")
    assert o.shape == q.shape and (o[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("L", [2, 5, 20])
def test_several_tokens(gpu_device, L, causal, dt):
    """Of sequences shorter than the tokens too: the first ones then see nothing."""
    from memory_amd.decode import paged_attention
    cache, dense = pool(gpu_device, dt, [0, 3, L, 64, 200], 16, 2, 64)
    q = torch.randn(5, L, 8, 64, generator=gen(2)).to(dt).to(gpu_device)
    o = paged_attention(q, cache, causal=causal)
    ref, bound = expect(q, dense, causal)
    ca.close(o, ref, bound, "out")
    assert (o[0] == 0).all() and (not causal or L <= 3 or (o[1, :L - 3] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 70])
def test_long(gpu_device, B):
    """Keys split over workgroups (one sequence) and not (many)."""
    from memory_amd.decode import paged_attention
    lens = [4000 - 37 * b for b in range(B)]
    cache, dense = pool(gpu_device, BF, lens, 64, 12 if B > 1 else 1, 64)
    q = torch.randn(B, 12, 64, generator=gen(3)).to(BF).to(gpu_device)
    ref, bound = expect(q[:, None], dense)
    ca.close(paged_attention(q, cache)[:, None], ref, bound, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 6])
def test_roomy_table(gpu_device, L):
    """A table with room for many times the tokens held: most workgroups find none."""
    from memory_amd.decode import PagedKVCache, paged_attention
    cache, dense = pool(gpu_device, BF, [90, 0, 7], 16, 2, 128)
    table = torch.full((3, 5000), -1, dtype=torch.int32, device=gpu_device)
    table[:, :cache.block_table.shape[1]] = cache.block_table
    roomy = PagedKVCache(cache.k_pages, cache.v_pages, table, cache.lengths)
    q = torch.randn(3, L, 8, 128, generator=gen(13)).to(BF).to(gpu_device)
    ref, bound = expect(q, dense, True)
    ca.close(paged_attention(q, roomy, causal=True), ref, bound, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1])
def test_entries_outside_the_pool(gpu_device, bad):
    """Keys of a page that is none do not count, and what is written there is dropped."""
    from memory_amd.decode import paged_attention
    lens = [100, 33]
    cache, dense = pool(gpu_device, BF, lens, 16, 2, 64, room=16)
    cache.block_table[0, 2] = bad
    cache.block_table[1, :] = bad
    holes = [torch.zeros(100, dtype=torch.bool, device=gpu_device), torch.ones(33, dtype=torch.bool, device=gpu_device)]
    holes[0][32:48] = True
    q = torch.randn(2, 1, 4, 64, generator=gen(4)).to(BF).to(gpu_device)
    o = paged_attention(q, cache)
    ref, bound = expect(q, dense, holes=holes)
    ca.close(o, ref, bound, "out")
    assert (o[1] == 0).all()
    before = cache.k_pages.clone(), cache.v_pages.clone()
    new = torch.ones(2, 1, 2, 64, device=gpu_device, dtype=BF)
    cache.append(new, new, positions=torch.tensor([40, 2], device=gpu_device))
    cache.append(new, new, positions=torch.tensor([-1, 10 ** 7], device=gpu_device))
    for a, b in zip(before, (cache.k_pages, cache.v_pages)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.gpu
def test_lengths_outside(gpu_device):
    """Lengths below 0 and past the table: none, and all of the table."""
    from memory_amd.decode import paged_attention
    cache, dense = pool(gpu_device, BF, [64, 64], 16, 1, 64)
    cache.lengths.copy_(torch.tensor([-5, 2 ** 31 - 1], dtype=torch.int32))
    q = torch.randn(2, 1, 2, 64, generator=gen(5)).to(BF).to(gpu_device)
    o = paged_attention(q, cache)
    ref, bound = expect(q, dense)
    ca.close(o[1:], ref[1:], bound[1:], "out")
    assert (o[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("treat", [False, True])
def test_append(gpu_device, treat, T, dt):
    """New rows land in their places (normed and rotated by place), everything else in the pool stays, lengths grow."""
    from memory_amd import ops
    lens = [0, 15, 16, 46]
    cache, _ = pool(gpu_device, dt, lens, 16, 2, 64, room=20)
    before = [cache.k_pages.clone(), cache.v_pages.clone()]
    g = gen(6)
    fused = torch.randn(4, T, 8, 64, generator=g).to(dt).to(gpu_device)
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(gpu_device)
    freq = ops.rope_frequencies(64, 10000.0, gpu_device)
    kw = dict(q=q, q_weight=w, k_weight=w * 2, inv_freq=freq) if treat else dict(q=q)
    pos = torch.tensor(lens, device=gpu_device)[:, None] + torch.arange(T, device=gpu_device)
    out = cache.append(k, v, **kw)
    assert cache.lengths.tolist() == [n + T for n in lens]
    if treat:
        for got, x, ww in ((out, q, w), (None, k, w * 2)):
            ref, bound = hr.reference(x, ww, 1e-6, True, pos, freq, False)
            if got is None:
                got = torch.stack([torch.stack([cache.k_pages[cache.block_table[b, p // 16], p % 16] for p in pos[b].tolist()])
                                   for b in range(4)])
            hr.close(got, ref, bound, "rows")
    else:
        assert torch.equal(out, q)
    for b in range(4):
        for i, p in enumerate(pos[b].tolist()):
            at = int(cache.block_table[b, p // 16]), p % 16
            assert torch.equal(cache.v_pages[at], v[b, i])
            if not treat:
                assert torch.equal(cache.k_pages[at], k[b, i])
            before[0][at], before[1][at] = cache.k_pages[at], cache.v_pages[at]
    for a, b in zip(before, (cache.k_pages, cache.v_pages)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    # the same places again, given: the same rows, and lengths stay
    was = cache.lengths.clone()
    again = cache.append(k, v, positions=pos[:, 0].int(), **kw)
    assert torch.equal(again, out) and torch.equal(was, cache.lengths)


@pytest.mark.gpu
def test_strided_pool(gpu_device):
    """K and V as halves of one pool, pages apart."""
    from memory_amd.decode import PagedKVCache, paged_attention
    g = gen(7)
    both = torch.randn(12, 2, 32, 2, 64, generator=g).to(BF).to(gpu_device)
    table = torch.tensor([[3, 7, 0], [11, 2, 5]], dtype=torch.int32, device=gpu_device)
    cache = PagedKVCache(both[:, 0], both[:, 1], table, torch.tensor([90, 41], dtype=torch.int32, device=gpu_device))
    dense = [(both[table[b].long(), 0].flatten(0, 1)[:n], both[table[b].long(), 1].flatten(0, 1)[:n]) for b, n in ((0, 90), (1, 41))]
    q = torch.randn(2, 4, 1, 64, generator=g).to(BF).to(gpu_device).transpose(1, 2)
    ref, bound = expect(q, dense)
    ca.close(paged_attention(q, cache), ref, bound, "out")


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu_device):
    """A pool of 2.2 G elements each for K and V; sequences at both ends of it."""
    from memory_amd.decode import PagedKVCache, paged_attention
    P, page, HK, D = 33600, 64, 8, 128
    k, v = (torch.empty(P, page, HK, D, device=gpu_device, dtype=BF) for _ in range(2))
    table = torch.tensor([[P - 1, 0, P - 2], [1, P - 3, P // 2]], dtype=torch.int32, device=gpu_device)
    g = torch.Generator(device=gpu_device).manual_seed(8)
    for i in table.flatten().tolist():
        k[i].normal_(generator=g)
        v[i].normal_(generator=g)
    cache = PagedKVCache(k, v, table, torch.tensor([150, 191], dtype=torch.int32, device=gpu_device))
    new = torch.randn(2, 1, HK, D, device=gpu_device, generator=g).to(BF)
    cache.append(new, new)
    assert torch.equal(k[P - 2, 150 - 128], new[0, 0]) and torch.equal(k[P // 2, 191 - 128], new[1, 0])
    dense = [(k[table[b].long()].flatten(0, 1)[:n], v[table[b].long()].flatten(0, 1)[:n]) for b, n in ((0, 151), (1, 192))]
    q = torch.randn(2, 1, 32, D, device=gpu_device, generator=g).to(BF)
    ref, bound = expect(q, dense)
    ca.close(paged_attention(q, cache), ref, bound, "out")


@pytest.mark.gpu
def test_captured_generation(gpu_device):
    """A captured step (append, attention) replayed while sequences grow over page borders gives the eager bits."""
    from memory_amd import ops
    from memory_amd.decode import PagedKVCache, paged_attention
    freq = ops.rope_frequencies(64, 10000.0, gpu_device)
    w = torch.ones(64, device=gpu_device)
    qkv = torch.zeros(3, 1, 8, 64, device=gpu_device, dtype=BF)

    def fresh():
        c = PagedKVCache.allocate(24, 16, 2, 64, 3, 8, device=gpu_device)
        c.block_table.copy_(torch.arange(24, dtype=torch.int32).view(8, 3).t())
        c.lengths.copy_(torch.tensor([0, 14, 30], dtype=torch.int32))
        return c

    def step(c):
        q = c.append(qkv[:, :, 4:6], qkv[:, :, 6:], q=qkv[:, :, :4], q_weight=w, k_weight=w, inv_freq=freq)
        return paged_attention(q, c, causal=True)

    a, b = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    a.lengths.copy_(b.lengths)
    for rep in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=gen(40 + rep)).to(BF))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step(b)), f"token {rep}"
        assert torch.equal(a.lengths, b.lengths) and torch.equal(a.k_pages, b.k_pages)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(qk_norm=True, rotary_dim=32)])
def test_layer_served(gpu_device, kw):
    """memory_decode_step over an encoder's states equals the module's forward: both project with the same weights, and
    attend within the bounds of the operators (float32: 1e-5 of the largest value is 40 times 2^-22)."""
    from memory_amd.decode import PagedKVCache, memory_decode_step
    m = ca._module(gpu_device, **kw)
    if kw:
        with torch.no_grad():
            m.k_norm.weight.mul_(1.5)
    h = torch.randn(3, 4, 256, generator=gen(9)).to(gpu_device)
    mem = torch.randn(3, 50, 96, generator=gen(10)).to(gpu_device)
    lens = torch.tensor([50, 0, 17], device=gpu_device)
    pos = dict(query_positions=torch.arange(4, device=gpu_device) + 9) if kw else {}
    with torch.no_grad():
        ref, _ = m(h, mem, memory_lengths=lens, **pos)
        cache = PagedKVCache.from_memory(m, mem, lens, page_size=16)
        at = dict(positions=pos["query_positions"]) if kw else {}
        whole = memory_decode_step(m, h, cache, **at)
        assert (whole - ref).abs().max() <= 1e-5 * ref.abs().max()
        for t in range(4):
            at = dict(positions=pos["query_positions"][t:t + 1]) if kw else {}
            one = memory_decode_step(m, h[:, t:t + 1], cache, **at)
            assert (one - ref[:, t:t + 1]).abs().max() <= 1e-5 * ref.abs().max()


@pytest.mark.gpu
def test_trained_and_served(gpu_device):
    """All of it in one run: a bfloat16 sublayer trained a few steps over ragged states, then served token by token."""
    from memory_amd.decode import PagedKVCache, memory_decode_step
    from memory_amd.memory_block import MemorySublayer
    torch.manual_seed(2)
    s = MemorySublayer(256, 4, 2, memory_dim=128, wo_init_zero=False, qk_norm=True, rotary_dim=64).to(gpu_device).to(BF)
    opt = torch.optim.AdamW(s.parameters(), lr=1e-3)
    h = torch.randn(4, 70, 256, generator=gen(11)).to(gpu_device).to(BF)
    mem = torch.randn(4, 91, 128, generator=gen(12)).to(gpu_device).to(BF)
    lens = torch.tensor([91, 3, 64, 0], device=gpu_device)
    for _ in range(3):
        opt.zero_grad()
        s(h, mem, memory_lengths=lens).float().square().mean().backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in s.parameters())
        opt.step()
    with torch.no_grad():
        ref = s(h, mem, memory_lengths=lens)
        cache = PagedKVCache.from_memory(s.memory_attn, mem, lens)
        x = s.memory_layernorm(h[:, 5:6])
        out = h[:, 5:6] + memory_decode_step(s.memory_attn, x, cache, positions=torch.tensor([5], device=gpu_device))
        # (two bfloat16 paths with their own roundings of queries, attention, projection and sum: 6 half steps)
        assert (out.float() - ref[:, 5:6].float()).abs().max() <= 6 * 2.0 ** -8 * ref.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("pages,most", [(4, 0), (0, 0), (0, 2)])
def test_append_without_places(gpu_device, pages, most, positions, dt):
    """A table without columns, a pool without pages: every token is dropped (three sequences of two tokens, so that rows
    in a piece would stay within the four pages), the queries are treated and lengths grow."""
    from memory_amd.decode import PagedKVCache, paged_attention
    g = gen(50)
    k, v = (torch.full((pages, 16, 2, 64), 7.0, device=gpu_device, dtype=dt) for _ in range(2))
    cache = PagedKVCache(k, v, torch.zeros(3, most, device=gpu_device, dtype=torch.int32),
                         torch.tensor([0, 1, 5], device=gpu_device, dtype=torch.int32))
    new = torch.randn(3, 2, 8, 64, generator=g).to(dt).to(gpu_device)
    q = cache.append(new[:, :, 4:6], new[:, :, 6:], q=new[:, :, :4],
                     positions=torch.zeros(3, device=gpu_device, dtype=torch.int64) if positions else None)
    assert torch.equal(q, new[:, :, :4]) and (k == 7).all() and (v == 7).all()
    assert cache.lengths.tolist() == ([0, 1, 5] if positions else [2, 3, 7])
    assert cache.append(new[:, :, 4:6], new[:, :, 6:], positions=cache.lengths) is None and (k == 7).all() and (v == 7).all()
    o = paged_attention(q, cache, causal=True)
    assert o.shape == q.shape and (o == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("L", [1, 5, 20])
@pytest.mark.parametrize("page,pages", [(16, 4), (48, 3)])
def test_causal_past_the_table(gpu_device, page, pages, L, dt):
    """Lengths past the table's end, as an append leaves them that dropped tokens: token l of L sees the places below
    lengths - L + l + 1 that there are, the same with room left in the table as without."""
    from memory_amd.decode import PagedKVCache, paged_attention
    room = page * pages
    lens = [room + n for n in (3, L, L + 7, -1, 0)] + [2 ** 31 - 1]
    cache, dense = pool(gpu_device, dt, [room] * len(lens), page, 2, 64)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.randn(len(lens), L, 8, 64, generator=gen(51)).to(dt).to(gpu_device)
    o = paged_attention(q, cache, causal=True)
    for b, n in enumerate(lens):
        k, v = dense[b]
        for l in range(L):
            see = min(room, n - L + l + 1)
            ref, bound = ca.reference(q[b:b + 1, l:l + 1], k[None, :see], v[None, :see])
            ca.close(o[b:b + 1, l:l + 1], ref, bound, f"length {n}, token {l}")
    roomy = torch.full((len(lens), pages + 3), -1, dtype=torch.int32, device=gpu_device)
    roomy[:, :pages] = cache.block_table
    cache.lengths[-1] = room + 40
    same = PagedKVCache(cache.k_pages, cache.v_pages, roomy, cache.lengths)
    # (other splits of the keys: the sums differ by their order)
    for b, n in enumerate(cache.lengths.tolist()):
        for l in range(L):
            see = min(room, n - L + l + 1)
            ref, bound = ca.reference(q[b:b + 1, l:l + 1], dense[b][0][None, :see], dense[b][1][None, :see])
            ca.close(paged_attention(q, same, causal=True)[b:b + 1, l:l + 1], ref, bound, f"with room, length {n}, token {l}")


@pytest.mark.gpu
def test_append_past_the_table(gpu_device):
    """A sequence of 62 tokens with room for 64 takes five more: two find a place, and each of the five sees itself where
    it has one and everything before it."""
    from memory_amd.decode import paged_attention
    cache, dense = pool(gpu_device, BF, [62], 16, 2, 64)
    new = torch.randn(1, 5, 12, 64, generator=gen(52)).to(BF).to(gpu_device)
    q = cache.append(new[:, :, 8:10], new[:, :, 10:], q=new[:, :, :8])
    assert cache.lengths.tolist() == [67]
    o = paged_attention(q, cache, causal=True)
    k, v = (torch.cat([d, x[0, :2]]) for d, x in zip(dense[0], (new[:, :, 8:10], new[:, :, 10:])))
    for l in range(5):
        see = min(64, 63 + l)
        ref, bound = ca.reference(q[:, l:l + 1], k[None, :see], v[None, :see])
        ca.close(o[:, l:l + 1], ref, bound, f"token {l}")


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(qk_norm=True, rotary_dim=32)])
def test_float16_layer_served(gpu_device, kw):
    """A float16 module, served from float32 pages, equals its forward: keys and queries are the same float16 values in
    both; the attention, float32 within 1e-5 of the largest value as in test_layer_served, is rounded to float16 in
    both, and a row of o_proj adds 256 such differences (2^-11 each, half a step on either side, against o_proj's own
    weights) before it is rounded itself."""
    from memory_amd.decode import PagedKVCache, memory_decode_step
    m = ca._module(gpu_device, dt=torch.float16, **kw)
    h = torch.randn(3, 4, 256, generator=gen(53)).half().to(gpu_device)
    mem = torch.randn(3, 50, 96, generator=gen(54)).half().to(gpu_device)
    lens = torch.tensor([50, 0, 17], device=gpu_device)
    pos = torch.arange(4, device=gpu_device) + 9 if kw else None
    with torch.no_grad():
        ref, _ = m(h, mem, memory_lengths=lens, query_positions=pos)
        cache = PagedKVCache.from_memory(m, mem, lens, page_size=16)
        assert cache.dtype == F32
        k, v = m.project_memory(mem)
        assert torch.equal(cache.k_pages[cache.block_table[0, 3], :2], k[0, 48:].float())
        assert torch.equal(cache.v_pages[cache.block_table[2, 1], :1], v[2, 16:17].float())
        whole = memory_decode_step(m, h, cache, positions=pos)
        assert whole.dtype == torch.float16 and (whole[1] == 0).all()
        a = m.attention_preproj(h, mem, memory_lengths=lens, query_positions=pos).double()
        slack = (2 * 2.0 ** -11 * a.abs() + 1e-5 * a.abs().max()) @ m.o_proj.weight.double().abs().t().contiguous()
        bound = slack + 2 * 2.0 ** -11 * ref.double().abs() + 2.0 ** -24
        assert ((whole.double() - ref.double()).abs() <= bound).all()
        for t in range(4):
            one = memory_decode_step(m, h[:, t:t + 1], cache, positions=None if pos is None else pos[t:t + 1])
            assert ((one.double() - ref[:, t:t + 1].double()).abs() <= bound[:, t:t + 1]).all()
