"""The 8-bit cache as a serving loop uses it: Kv8Cache over ragged prompts, decode steps (all of the context, and chosen
pages), roll-backs and reused pages, eager and captured; the model with it."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
import serving_ref
from lucciola_rs_amd.engine import Kv8Cache, RopeCache, sm_scale
from lucciola_rs_amd.model import Qwen2Config, Qwen2Model, random_weights

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def held(cache, ids, layer):
    """float64 K and V [16 pages, hkv, d] that pages of a cache hold."""
    out = []
    for is_v, pool in enumerate((cache.k_pool, cache.v_pool)):
        codes = ref.TABLE[pool[ids, layer].cpu().numpy()]
        d = cache.head_dim
        codes = codes.reshape(*codes.shape[:2], 4, d, 4).swapaxes(-1, -2).reshape(*codes.shape[:2], PAGE, d) if is_v else \
            codes.reshape(*codes.shape[:2], PAGE, d)
        val = codes * cache.scales[ids, layer, :, is_v].cpu().numpy().astype(np.float64)[..., None, None]
        out.append(torch.from_numpy(np.ascontiguousarray(val.swapaxes(1, 2))).view(-1, val.shape[1], d).cuda())
    return out


class Loop:
    """A Kv8Cache, and every sequence's exact K and V (float64, as they were appended)."""

    def __init__(self, luc, seqs, pages, max_pos, hq, hkv, d, dtype, norm, bias, layers=2, max_rows=700):
        gen = torch.Generator().manual_seed(d + hq)
        rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.hq, self.hkv, self.d, self.dt, self.layers, self.gen = hq, hkv, d, DT[dtype], layers, gen
        self.cache = Kv8Cache(layers, hq, hkv, d, pages, seqs, max_pos, max_rows, bounds=True, lib=luc)
        # whatever pages hold before a sequence gets them
        self.cache.k_pool.fill_(0xFF)
        self.cache.v_pool.fill_(0x7F)
        self.cache.scales.fill_(2.0 ** 8)
        self.cache.bounds.fill_(0x7E)
        self.rope = RopeCache(max_pos, d, lib=luc)
        self.maps = serving_ref.Maps(seqs, self.cache.blocks.block_tables.shape[1], pages)
        width = (hq + 2 * hkv) * d
        a, b = hq * d, (hq + hkv) * d
        self.kw = {}
        if bias:
            x = (rnd(width) * 0.3).to(self.dt).cuda()
            self.kw.update(q_bias=x[:a], k_bias=x[a:b], v_bias=x[b:])
        if norm:
            self.kw.update(q_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda(), k_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda())
        self.exact = [[([], []) for _ in range(layers)] for _ in range(seqs)]
        # the largest that a page of a sequence has seen, for its scale: a roll-back does not take it back
        self.top = np.zeros((pages, layers, hkv, 2))

    def rows(self, n):
        return (torch.randn(n, (self.hq + 2 * self.hkv) * self.d, generator=self.gen) * 1.4).to(self.dt).cuda()

    def split(self, qkv):
        a, b = self.hq * self.d, (self.hq + self.hkv) * self.d
        return qkv[:, :a], qkv[:, a:b], qkv[:, b:]

    def truncate(self, keep):
        self.cache.truncate(i32(keep))
        self.maps.truncate(keep)
        for b, k in enumerate(keep):
            for xs in (x for layer in self.exact[b] for x in layer):
                del xs[k:]

    def step(self, new, max_rows=None, budget=None):
        """One step of every layer, checked against 64 bits; budget: of chosen pages."""
        total = sum(new)
        slots, positions, cu, start = self.maps.extend(new)
        self.cache.extend(i32(new), rows=total)
        blocks = self.cache.blocks
        assert blocks.slots[:total].tolist() == slots and blocks.positions[:total].tolist() == positions
        max_ctx = max(self.maps.lens)
        print(f"  step: new {new}, held {start}, budget {budget}", flush=True)
        for layer in range(self.layers):
            qkv = self.rows(total)
            q, k, v = self.split(qkv)
            want, terms = [], []
            cos, sin = self.rope.cos[positions], self.rope.sin[positions]
            for x, heads, name in ((q, self.hq, "q"), (k, self.hkv, "k")):
                bias = self.kw.get(f"{name}_bias")
                y, t = serving_ref.norm_rope(x.view(total, heads, self.d), None if bias is None else bias.view(heads, self.d),
                                             self.kw.get(f"{name}_norm"), 1e-6, cos, sin)
                want.append(y)
                terms.append(t)
            exact_v = v.double() + (self.kw["v_bias"].double() if "v_bias" in self.kw else 0)
            exact_v = exact_v.view(total, self.hkv, self.d)
            for r, s in enumerate(slots):
                if s % PAGE == 0:
                    self.top[s // PAGE, layer] = 0
                for is_v, x in ((0, want[1]), (1, exact_v)):
                    at = self.top[s // PAGE, layer, :, is_v]
                    np.maximum(at, x[r].abs().amax(-1).cpu().numpy(), out=at)
            for b in range(len(new)):
                self.exact[b][layer][0].extend(want[1][cu[b]:cu[b + 1]])
                self.exact[b][layer][1].extend(exact_v[cu[b]:cu[b + 1]])
            k_tol = float(serving_ref.append_tolerance(want[1], terms[1], self.dt).max())
            out = torch.full((total, self.hq * self.d), 7.0, dtype=self.dt, device="cuda")
            self.cache.append(layer, q, k, v, self.rope, **self.kw)
            err = (q.double().view_as(want[0]) - want[0]).abs()
            assert bool((err <= serving_ref.append_tolerance(want[0], terms[0], self.dt)).all())
            pages = None
            if budget is None:
                self.cache.attend(layer, out, q, max_ctx, max_rows)
            else:
                pages = self.cache.attend_sparse(layer, out, q, max_ctx, budget)
            for b, n in enumerate(new):
                if n:
                    self.check_sequence(b, layer, q[cu[b]:cu[b + 1]], out[cu[b]:cu[b + 1]], start[b], k_tol,
                                        None if pages is None else pages[b])
                elif pages is not None:
                    assert bool((pages[b] == -1).all())
        blocks.check()
        assert blocks.num_free == len(self.maps.free)

    def check_sequence(self, b, layer, q, out, start, k_tol, pages):
        ctx = self.maps.lens[b]
        ids = self.maps.tables[b, :-(-ctx // PAGE)].astype(np.int64)
        values = held(self.cache, ids, layer)
        slots = torch.from_numpy((ids[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:ctx]).cuda()
        reads = [torch.zeros(ctx, self.hkv * self.d, dtype=self.dt, device="cuda") for _ in range(2)]
        self.cache.read(layer, *reads, slots)
        for is_v, (val, got) in enumerate(zip(values, reads)):
            val = val[:ctx]
            assert torch.equal(got, val.reshape(ctx, -1).to(self.dt))
            exact = torch.stack(self.exact[b][layer][is_v])
            # half a step of e4m3, 2^-4 of the value, and of its subnormals, 2^-10 of the scale, once when it is
            # stored and again (of the subnormals) whenever the scale grows, 8 times at most here; the scale is below
            # 2 / 448 of the page's largest value; the 16-bit value's own rounding
            top = torch.from_numpy(self.top[ids, layer, :, is_v]).cuda().repeat_interleave(PAGE, 0)[:ctx, :, None]
            fi = torch.finfo(self.dt)
            room = 2.0 ** -4 * exact.abs() + 9 * 2.0 ** -10 * (2 / 448) * top + fi.eps * exact.abs() + (0 if is_v else k_tol)
            assert bool(((val - exact).abs() <= room * (1 + 2.0 ** -4)).all()), (b, layer, is_v)
        n, g = q.shape[0], self.hq // self.hkv
        pos = torch.arange(ctx, device="cuda")
        seen = pos[None] <= (start + torch.arange(n, device="cuda"))[:, None]
        for h in range(self.hkv):
            heads = slice(h * g, (h + 1) * g)
            view = seen
            if pages is not None:
                want = ref.choose(ref.scores(q[0].double().cpu().numpy().reshape(self.hq, self.d)[heads],
                                             self.cache.bounds[ids, layer, h].cpu().numpy(),
                                             self.cache.scales[ids, layer, h, 0].cpu().numpy()), pages.shape[-1], 1, 2)
                assert pages[h].tolist() == want
                view = seen & torch.isin(pos // PAGE, pages[h])[None]
            want, tol = ref.attention(q.double().view(n, self.hq, self.d)[:, heads], *(x[:ctx, h:h + 1] for x in values), view,
                                      sm_scale(self.d), self.dt)
            serving_ref.check(out.view(n, self.hq, self.d)[:, heads], want, tol, self.dt, f"layer {layer} sequence {b} head {h}")


@pytest.mark.parametrize("hq,hkv,d,dtype,norm,bias", [(14, 2, 64, "f16", True, False), (12, 2, 128, "bf16", False, True),
                                                      (8, 8, 64, "bf16", True, True), (5, 1, 128, "f16", False, False)])
def test_a_serving_loop(luc, hq, hkv, d, dtype, norm, bias):
    """Prompts, decode steps, a chunk beside them, roll-backs, a sequence that ends and one that
    takes its pages."""
    loop = Loop(luc, 4, 60, 512, hq, hkv, d, dtype, norm, bias)
    loop.step([37, 0, 300, 16])
    loop.step([1, 0, 1, 1])
    loop.step([1, 0, 1, 1], budget=8)
    loop.step([1, 5, 1, 1], max_rows=5)
    loop.truncate([20, 512, 299, 0])     # a rejected draft, one row less, an end
    loop.step([1, 1, 1, 1], budget=3)
    loop.step([130, 1, 0, 61])
    loop.truncate([0, 0, 0, 0])
    assert loop.cache.blocks.num_free == 60
    loop.step([0, 511, 0, 33])
    loop.step([0, 1, 0, 1], budget=20)
    loop.step([0, 0, 0, 1])


def test_a_captured_step_against_an_eager_twin(luc):
    """One graph of a whole decode step (pages, three layers, one of them over chosen pages, a roll-back of one
    sequence at every replay) replayed with eager work between, against the same calls made eagerly on another cache."""
    hq, hkv, d, seqs, layers, budget = 12, 2, 128, 3, 3, 9
    caches = [Kv8Cache(layers, hq, hkv, d, 64, seqs, 320, 200, bounds=True, lib=luc) for _ in range(2)]
    rope = RopeCache(320, d, lib=luc)
    gen = torch.Generator().manual_seed(3)
    width = (hq + 2 * hkv) * d
    rnd = lambda n: (torch.randn(n, width, generator=gen) * 1.4).to(torch.bfloat16).cuda()  # noqa: E731

    def layer_calls(cache, layer, qkv, out, max_rows):
        q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        cache.append(layer, q, k, v, rope)
        if layer == 1 and max_rows == 1:
            cache.attend_sparse(layer, out, q, 320, budget)
        else:
            cache.attend(layer, out, q, 320, max_rows)

    for layer_rows in [[rnd(245) for _ in range(layers)]]:
        for c in caches:
            c.blocks.max_rows = 245
            c.blocks.slots = torch.full((245,), -1, dtype=torch.int64, device="cuda")
            c.blocks.positions = torch.full((245,), -1, dtype=torch.int32, device="cuda")
            c.extend(i32([165, 15, 65]), rows=245)
            for layer, qkv in enumerate(layer_rows):
                layer_calls(c, layer, qkv.clone(), torch.empty(245, hq * d, dtype=torch.bfloat16, device="cuda"), 165)
    one = i32([1] * seqs)
    keep = i32([320, 14, 320])
    qkv_in = [rnd(seqs) for _ in range(layers)]
    outs = [torch.zeros(seqs, hq * d, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]

    def step(cache, qkvs, outs):
        cache.truncate(keep)
        cache.extend(one, rows=seqs)
        for layer in range(layers):
            layer_calls(cache, layer, qkvs[layer], outs[layer], 1)

    caches[0].workspace(seqs, 1, 320)
    caches[0].workspace(seqs, 1, 320, budget)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    held_in = [x.clone() for x in qkv_in]
    with torch.cuda.graph(graph):
        for a, b in zip(held_in, qkv_in):  # (append rotates q in place)
            a.copy_(b)
        step(caches[0], held_in, outs)
    for _ in range(40):
        fresh = [rnd(seqs) for _ in range(layers)]
        for a, b in zip(qkv_in, fresh):
            a.copy_(b)
        graph.replay()
        eager = [torch.zeros_like(o) for o in outs]
        step(caches[1], [x.clone() for x in fresh], eager)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b) and bool(a.isfinite().all())
    assert caches[0].blocks.lens.tolist() == [205, 15, 105]
    for name in ("k_pool", "v_pool", "scales", "bounds"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    caches[0].blocks.check()


def test_a_workspace_is_made_before_a_capture(luc):
    cache = Kv8Cache(1, 8, 2, 64, 400, 1, 6000, bounds=True, lib=luc)
    q = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    for call in (lambda: cache.attend(0, torch.empty_like(q), q, 6000), lambda: cache.attend_sparse(0, torch.empty_like(q), q, 6000, 50)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(graph):
                q.add_(0)
                call()
    ws = cache.workspace(1, 1, 6000)
    assert cache.workspace(1, 1, 1000) in (None, ws) and cache.workspace(1, 1, 6000, 50) is not None


def test_two_streams_at_once(luc):
    """Steps of two caches on two streams that overlap, with a workspace each: the bits of the same
    steps in turn."""
    hq, hkv, d, steps, budget = 14, 2, 64, 12, 30
    rope = RopeCache(3000, d, lib=luc)
    width = (hq + 2 * hkv) * d

    def prepare(seed):
        gen = torch.Generator().manual_seed(seed)
        cache = Kv8Cache(1, hq, hkv, d, 400, 2, 3000, 2700, bounds=True, lib=luc)
        rnd = lambda n: (torch.randn(n, width, generator=gen) * 1.4).half().cuda()  # noqa: E731
        work = [(i32([1500 + 100 * seed, 900]), rnd(2400 + 100 * seed), 1700)] + [(i32([1, 1]), rnd(2), 1) for _ in range(steps)]
        for args in ((2, 1, 3000), (2, 1, 3000, budget), (2400 + 100 * seed, 1700, 3000)):
            cache.workspace(*args)
        return cache, work, [torch.zeros(w.shape[0], hq * d, dtype=torch.float16, device="cuda") for _, w, _ in work]

    def issue(cache, work, outs, i, stream):
        new, qkv, most = work[i]
        cache.extend(new, rows=qkv.shape[0], stream=stream)
        q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        cache.append(0, q, k, v, rope, stream=stream)
        if i % 2:
            cache.attend_sparse(0, outs[i], q, 3000, budget, stream=stream)
        else:
            cache.attend(0, outs[i], q, 3000, most, stream=stream)

    results = []
    for together in (False, True):
        sets = [prepare(seed) for seed in (1, 2)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets] if together else [None, None]
        for i in range(steps + 1):
            for (cache, work, outs), stream in zip(sets, streams):
                issue(cache, work, outs, i, stream)
        torch.cuda.synchronize()
        for cache, _, _ in sets:
            cache.blocks.check()
        results.append([o for _, _, outs in sets for o in outs])
    for a, b in zip(*results):
        assert torch.equal(a, b) and bool(a.isfinite().all())


# ---- the model ------------------------------------------------------------------------------

CFG = Qwen2Config(vocab_size=512, hidden_size=256, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                  intermediate_size=512, max_position_embeddings=512)


@pytest.fixture(scope="module", params=[0, 4], ids=["dense", "sparse"])
def model(luc, request):
    return Qwen2Model(CFG, random_weights(CFG, seed=5, std=0.05), lib=luc, kv_format="e4m3", sparse_pages=request.param)


def test_model_attention_is_that_of_its_cache(luc, model):
    """forward() of a prompt, single tokens, a second chunk and a step back: every layer's attention
    against 64 bits over what the cache holds."""
    d, hq, hkv = CFG.head_dim, CFG.num_attention_heads, CFG.num_key_value_heads
    g = hq // hkv
    calls = []
    inner = model.kv.attend, model.kv.attend_sparse

    def attend(layer, out, q, max_ctx, *rest, **kw):
        inner[0](layer, out, q, max_ctx, *rest, **kw)
        calls.append((layer, out.clone(), q.clone(), max_ctx, None))

    def attend_sparse(layer, out, q, max_ctx, budget, *rest, **kw):
        pages = inner[1](layer, out, q, max_ctx, budget, *rest, **kw)
        assert budget == model.sparse_pages
        calls.append((layer, out.clone(), q.clone(), max_ctx, pages.clone()))
        return pages

    model.kv.attend, model.kv.attend_sparse = attend, attend_sparse
    try:
        rng = np.random.default_rng(2)
        for n, pos in ((40, 0), (1, 40), (1, 41), (70, 42), (1, 112), (2, 30), (1, 32)):
            calls.clear()
            model.forward(rng.integers(0, CFG.vocab_size, n).tolist(), pos)
            assert len(calls) == CFG.num_hidden_layers and int(model.kv.blocks.lens) == pos + n
            ids = model.kv.blocks.block_tables[0, :-(-(pos + n) // PAGE)].cpu().numpy().astype(np.int64)
            for layer, out, q, ctx, pages in calls:
                assert ctx == pos + n and (pages is not None) == bool(model.sparse_pages and n == 1)
                values = [x[:ctx] for x in held(model.kv, ids, layer)]
                at = torch.arange(ctx, device="cuda")
                seen = at[None] <= (pos + torch.arange(n, device="cuda"))[:, None]
                for h in range(hkv):
                    view = seen if pages is None else seen & torch.isin(at // PAGE, pages[0, h])[None]
                    heads = slice(h * g, (h + 1) * g)
                    want, tol = ref.attention(q.double().view(n, hq, d)[:, heads], *(x[:, h:h + 1] for x in values), view,
                                              sm_scale(d), torch.bfloat16)
                    serving_ref.check(out.view(n, hq, d)[:, heads], want, tol, torch.bfloat16, f"{n} rows at {pos}, layer {layer}")
            assert bool(model.logits().isfinite().all())
    finally:
        del model.kv.attend, model.kv.attend_sparse


def test_model_graph_replays_the_eager_loop(luc, model):
    """capture_decode over an 8-bit cache: the eager loop's tokens, twice from the same prompt (contexts
    below one split: the same arithmetic)."""
    prompt = np.random.default_rng(8).integers(0, CFG.vocab_size, 70).tolist()
    model.forward(prompt, 0)
    eager, pos = [model.sample_greedy()], len(prompt)
    for _ in range(24):
        model.forward([eager[-1]], pos)
        eager.append(model.sample_greedy())
        pos += 1
    graph = model.capture_decode(max_ctx=256)
    for _ in range(2):
        model.forward(prompt, 0)
        assert model.sample_greedy() == eager[0]
        model.pos.fill_(len(prompt))
        for s in range(24):
            graph.replay()
            assert int(model.idx) == eager[s + 1], s
        assert int(model.kv.blocks.lens) == int(model.pos) == len(prompt) + 24
    # eager again, from a step of the graph's
    model.forward([eager[9]], len(prompt) + 9)
    assert model.sample_greedy() == eager[10]
    model.kv.blocks.check()


def test_model_refusals(luc):
    w = random_weights(CFG, seed=5)
    for kw, text in ((dict(kv_format="e5m2"), "kv_format 'e5m2'"), (dict(kv_format="e4m3", kv_bits=4), "kv_format 'e4m3'"),
                     (dict(sparse_pages=8), "sparse_pages 8"), (dict(kv_bits=4, sparse_pages=8), "sparse_pages 8"),
                     (dict(kv_format="e4m3", sparse_pages=2), "sparse_pages 2")):
        with pytest.raises(ValueError, match=text):
            Qwen2Model(CFG, w, lib=luc, **kw)
    small = Qwen2Model(CFG, w, num_blocks=2, lib=luc, kv_format="e4m3")
    small.forward([1, 2, 3], 0)
    with pytest.raises(ValueError, match="past the 3 tokens of the 8-bit cache"):
        small.forward([4], 5)
    with pytest.raises(RuntimeError, match="Out of memory blocks"):
        small.forward(list(range(33)), 0)
    with pytest.raises(RuntimeError, match="Out of memory blocks"):
        small.capture_decode(40)
