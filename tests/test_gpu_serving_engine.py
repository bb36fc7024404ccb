"""Kv4Cache over steps whose sizes change: workspaces that captured graphs hold, buffers of earlier steps."""
import weakref

import pytest
import torch

from lucciola_rs_amd.engine import Kv4Cache, RopeCache
from lucciola_rs_amd.model import Qwen2Config, Qwen2Model, random_weights

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rows_of(gen, n, hq, hkv, d, dt):
    qkv = (torch.randn(n, (hq + 2 * hkv) * d, generator=gen) * 1.4).to(dt).cuda()
    a, b = hq * d, (hq + hkv) * d
    return qkv[:, :a], qkv[:, a:b], qkv[:, b:]


def test_a_graph_keeps_its_workspace(luc):
    """A captured step's splits after the cache's workspace has grown past it and its like are reused."""
    hq, hkv, d, ctx = 12, 2, 128, 6000
    cache = Kv4Cache(1, hq, hkv, d, 800, 1, 8000, 6000, lib=luc)
    rope = RopeCache(8000, d, lib=luc)
    gen = torch.Generator().manual_seed(1)
    cache.extend(i32([ctx]), rows=ctx)
    cache.append(0, *rows_of(gen, ctx, hq, hkv, d, torch.bfloat16), rope)
    q = rows_of(gen, 1, hq, hkv, d, torch.bfloat16)[0].contiguous()
    blocks = cache.blocks
    blocks.cu_seqlens.copy_(i32([0, 1]))
    blocks.start_pos.fill_(ctx - 1)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    cache.attend(0, want, q, ctx)
    size = cache.workspace(1, 1, ctx).numel()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(0, out, q, ctx)
    assert cache.workspace(500, 500, 8000).numel() > size
    for i in range(4):
        junk = [torch.full((size,), float("nan"), device="cuda") for _ in range(4)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(bool(x.isnan().all()) for x in junk)


def test_a_padded_append_after_a_longer_step(luc):
    """A step of fewer rows than the one before it: an append of more of them is refused and writes nothing; one that
    the step has room for leaves what it has no rows for alone."""
    hq, hkv, d = 4, 2, 64
    cache = Kv4Cache(1, hq, hkv, d, 20, 2, 128, 100, lib=luc)
    rope = RopeCache(128, d, lib=luc)
    gen = torch.Generator().manual_seed(2)
    cache.extend(i32([60, 30]), rows=90)
    cache.append(0, *rows_of(gen, 90, hq, hkv, d, torch.float16), rope)
    was = cache.k_pool.clone(), cache.v_pool.clone()
    cache.extend(i32([1, 1]), rows=2)
    with pytest.raises(ValueError, match="the step has 2"):
        cache.append(0, *rows_of(gen, 8, hq, hkv, d, torch.float16), rope)
    assert torch.equal(cache.k_pool, was[0]) and torch.equal(cache.v_pool, was[1])
    cache.truncate(i32([60, 30]))
    cache.extend(i32([1, 1]), rows=8)  # rows for a batch padded to 8
    cache.append(0, *rows_of(gen, 8, hq, hkv, d, torch.float16), rope)
    slots = cache.blocks.slots[:8].tolist()
    assert slots[2:] == [-1] * 6
    changed = (cache.k_pool != was[0]).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {s // 16 for s in slots[:2]}
    cache.blocks.check()


def test_a_step_without_rows(luc):
    hq, hkv, d = 4, 2, 128
    cache = Kv4Cache(1, hq, hkv, d, 20, 2, 128, 100, lib=luc)
    rope = RopeCache(128, d, lib=luc)
    gen = torch.Generator().manual_seed(3)
    cache.extend(i32([40, 0]), rows=40)
    cache.append(0, *rows_of(gen, 40, hq, hkv, d, torch.bfloat16), rope)
    was = cache.k_pool.clone(), cache.v_pool.clone(), cache.blocks.free_list.clone()
    cache.extend(i32([0, 0]), rows=0)
    q, k, v = rows_of(gen, 0, hq, hkv, d, torch.bfloat16)
    cache.append(0, q, k, v, rope)
    cache.attend(0, torch.empty_like(q), q, 128)
    cache.blocks.check()
    assert cache.blocks.lens.tolist() == [40, 0] and cache.blocks.cu_seqlens.tolist() == [0, 0, 0]
    now = cache.k_pool, cache.v_pool, cache.blocks.free_list
    assert all(torch.equal(a, b) for a, b in zip(was, now))


def test_a_decode_graph_keeps_its_workspace(luc):
    """capture_decode over the 16-bit cache: the graph's split-K workspace outlives the cache's."""
    cfg = Qwen2Config(vocab_size=256, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      intermediate_size=512, max_position_embeddings=4096)
    model = Qwen2Model(cfg, random_weights(cfg, seed=6, std=0.05), lib=luc)
    prompt = [i * 7 % 256 for i in range(900)]
    model.forward(prompt, 0)
    graph = model.capture_decode(max_ctx=1024)
    ws = weakref.ref(model.kv._workspace)
    model.kv.workspace(cfg.num_attention_heads, 4096)
    assert ws() is not None and ws() is not model.kv._workspace
    want = None
    for _ in range(3):
        model.forward(prompt, 0)
        model.idx.fill_(5)
        model.pos.fill_(len(prompt))
        tokens = []
        for _ in range(8):
            junk = [torch.full((ws().numel(),), float("nan"), device="cuda") for _ in range(3)]
            graph.replay()
            tokens.append(int(model.idx))
            assert all(bool(x.isnan().all()) for x in junk)
        want = want or tokens
        assert tokens == want
    del graph
    assert ws() is None
