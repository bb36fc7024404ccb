"""Page maps, normed appends and attention together, as a serving loop uses them: Kv4Cache and
DeviceBlocks over ragged prompts, decode steps, roll-backs and reused pages, eager and captured; the
model with a 4-bit cache; and attention where its work splits change."""
import numpy as np
import pytest
import torch

import serving_ref as ref
from test_gpu_kv4_attention import Cache, run, verify
from lucciola_rs_amd import library
from lucciola_rs_amd.engine import DeviceBlocks, Kv4Cache, RopeCache, sm_scale
from lucciola_rs_amd.model import Qwen2Config, Qwen2Model, random_weights

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def unpack(pool, page_ids, layer, d, is_v):
    """float64 values [16 pages, heads, d] that pages of a 4-bit pool hold."""
    by = pool[page_ids, layer].cpu().numpy()
    n_by, sm = by[..., :8 * d], np.ascontiguousarray(by[..., 8 * d:]).view(np.float16)
    lead = by.shape[:-1]
    if is_v:
        n_by = n_by.reshape(*lead, 2, d // 4, 8, 2).swapaxes(-3, -2).reshape(*lead, PAGE, d // 2)
        sm = np.moveaxis(sm.reshape(*lead, 2, d // 32, 2, 8), -1, -3).reshape(*lead, PAGE, d // 32, 2)
    else:
        n_by = n_by.reshape(*lead, PAGE, d // 2)
        sm = sm.reshape(*lead, PAGE, d // 32, 2)
    n = np.stack([n_by & 15, n_by >> 4], -1).reshape(*lead, PAGE, d)
    val = ref.values(n, np.ascontiguousarray(sm[..., 0]), np.ascontiguousarray(sm[..., 1]))
    step = np.repeat(sm[..., 0].astype(np.float64), 32, -1)
    out = [np.ascontiguousarray(x.swapaxes(1, 2)).reshape(-1, lead[1], d) for x in (val, step)]
    return [torch.from_numpy(x).cuda() for x in out]


class Loop:
    """A Kv4Cache, and every sequence's exact K and V (float64, as they were appended)."""

    def __init__(self, luc, seqs, pages, max_pos, hq, hkv, d, dtype, norm, bias, layers=2, max_rows=700):
        gen = torch.Generator().manual_seed(d + hq)
        rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.hq, self.hkv, self.d, self.dt, self.layers, self.gen = hq, hkv, d, DT[dtype], layers, gen
        self.cache = Kv4Cache(layers, hq, hkv, d, pages, seqs, max_pos, max_rows, lib=luc)
        # whatever pages hold before a sequence gets them: NaN steps and minima
        self.cache.k_pool.fill_(0xFF)
        self.cache.v_pool.fill_(0xFF)
        self.rope = RopeCache(max_pos, d, lib=luc)
        self.maps = ref.Maps(seqs, self.cache.blocks.block_tables.shape[1], pages)
        width = (hq + 2 * hkv) * d
        a, b = hq * d, (hq + hkv) * d
        self.kw = {}
        if bias:
            x = (rnd(width) * 0.3).to(self.dt).cuda()
            self.kw.update(q_bias=x[:a], k_bias=x[a:b], v_bias=x[b:])
        if norm:
            self.kw.update(q_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda(), k_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda())
        self.exact = [[([], []) for _ in range(layers)] for _ in range(seqs)]

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

    def step(self, new, max_rows=None):
        """One step of every layer, checked against 64 bits."""
        total = sum(new)
        slots, positions, cu, start = self.maps.extend(new)
        self.cache.extend(i32(new), rows=total)
        blocks = self.cache.blocks
        assert blocks.slots[:total].tolist() == slots and blocks.positions[:total].tolist() == positions
        assert blocks.cu_seqlens.tolist() == cu and blocks.start_pos.tolist() == start
        max_ctx = max(self.maps.lens)
        print(f"  step: new {new}, held {start}", flush=True)
        for layer in range(self.layers):
            qkv = self.rows(total)
            q, k, v = self.split(qkv)
            want, terms = [], []
            cos, sin = self.rope.cos[positions], self.rope.sin[positions]
            for x, heads, name in ((q, self.hq, "q"), (k, self.hkv, "k")):
                bias = self.kw.get(f"{name}_bias")
                y, t = ref.norm_rope(x.view(total, heads, self.d), None if bias is None else bias.view(heads, self.d),
                                     self.kw.get(f"{name}_norm"), 1e-6, cos, sin)
                want.append(y)
                terms.append(t)
            exact_v = v.double() + (self.kw["v_bias"].double() if "v_bias" in self.kw else 0)
            exact_v = exact_v.view(total, self.hkv, self.d)
            for b in range(len(new)):
                self.exact[b][layer][0].extend(want[1][cu[b]:cu[b + 1]])
                self.exact[b][layer][1].extend(exact_v[cu[b]:cu[b + 1]])
            k_tol = float(ref.append_tolerance(want[1], terms[1], self.dt).max())
            out = torch.full((total, self.hq * self.d), 7.0, dtype=self.dt, device="cuda")
            self.cache.append(layer, q, k, v, self.rope, **self.kw)
            err = (q.double().view_as(want[0]) - want[0]).abs()
            assert bool((err <= ref.append_tolerance(want[0], terms[0], self.dt)).all())
            self.cache.attend(layer, out, q, max_ctx, max_rows)
            for b, n in enumerate(new):
                if n:
                    self.check_sequence(b, layer, q[cu[b]:cu[b + 1]], out[cu[b]:cu[b + 1]], start[b], k_tol)
        blocks.check()
        assert blocks.num_free == len(self.maps.free)

    def check_sequence(self, b, layer, q, out, start, k_tol):
        ctx = self.maps.lens[b]
        ids = self.maps.tables[b, :-(-ctx // PAGE)].astype(np.int64)
        held = []
        for pool, is_v, tol in ((self.cache.k_pool, False, k_tol), (self.cache.v_pool, True, 0.0)):
            val, s = (x[:ctx] for x in unpack(pool, ids, layer, self.d, is_v))
            exact = torch.stack(self.exact[b][layer][is_v])
            # half a step for n's rounding; 2^-11 of s times 15 and of m for theirs (the largest n s and m are
            # within 15 s + |value|); the 16-bit value's own rounding
            fi = torch.finfo(self.dt)
            room = s / 2 + 2.0 ** -10 * (15 * s + exact.abs()) + fi.eps * exact.abs() + tol
            assert bool(((val - exact).abs() <= room).all()), (b, layer, is_v)
            held.append(val)
        want, tol = ref.attention(q.double().view(-1, self.hq, self.d), *held, start, sm_scale(self.d))
        ref.check(out.view(-1, self.hq, self.d), want, tol, self.dt, f"layer {layer} sequence {b}")


@pytest.mark.parametrize("hq,hkv,d,dtype,norm,bias", [(14, 2, 64, "f16", True, False), (12, 2, 128, "bf16", False, True),
                                                      (8, 8, 64, "bf16", True, True), (5, 1, 128, "f16", False, False)])
def test_a_serving_loop(luc, hq, hkv, d, dtype, norm, bias):
    """Prompts, decode steps, a chunk beside them, roll-backs, a sequence that ends and one that
    takes its pages."""
    loop = Loop(luc, 4, 60, 512, hq, hkv, d, dtype, norm, bias)
    loop.step([37, 0, 300, 16])
    loop.step([1, 0, 1, 1])
    loop.step([1, 5, 1, 1], max_rows=5)
    loop.truncate([20, 512, 299, 0])     # a rejected draft, one row less, an end
    loop.step([1, 1, 1, 1])
    loop.step([130, 1, 0, 61])
    loop.truncate([0, 0, 0, 0])
    assert loop.cache.blocks.num_free == 60
    loop.step([0, 512, 0, 33])
    loop.step([0, 0, 0, 1])


def test_a_step_that_cannot_be_met(luc):
    """Too few pages, table entries or rows: nothing is taken, outputs stay, check() tells which and the
    loop goes on."""
    loop = Loop(luc, 2, 8, 96, 4, 2, 64, "f16", False, False, layers=1, max_rows=80)
    loop.step([40, 20])
    blocks = loop.cache.blocks
    for new, rows, code, text in (([40, 40], 80, -6, "free pages are short"), ([57, 0], 80, -1, "a block table row is"),
                                  ([3, 0], 2, -1, "more rows")):
        loop.cache.extend(i32(new), rows=rows)
        assert blocks.lens.tolist() == [40, 20] and blocks.cu_seqlens.tolist() == [0, 0, 0]
        qkv = loop.rows(rows)
        q, k, v = loop.split(qkv)
        was = loop.cache.k_pool.clone(), loop.cache.v_pool.clone()
        out = torch.full((rows, 4 * 64), 7.0, dtype=loop.dt, device="cuda")
        loop.cache.append(0, q, k, v, loop.rope)
        loop.cache.attend(0, out, q, 96, 57)
        assert bool((out == 7).all())
        assert torch.equal(loop.cache.k_pool, was[0]) and torch.equal(loop.cache.v_pool, was[1])
        with pytest.raises(library.LucError, match=text) as e:
            blocks.check()
        assert e.value.code == code
        blocks.check()
    loop.step([1, 44])
    loop.step([1, 0])


def test_a_captured_step_against_an_eager_twin(luc):
    """One graph of a whole decode step (pages, three layers, a roll-back of one sequence at every replay)
    replayed with eager work between, against the same calls made eagerly on another cache."""
    hq, hkv, d, seqs, layers = 12, 2, 128, 3, 3
    caches = [Kv4Cache(layers, hq, hkv, d, 64, seqs, 320, 200, lib=luc) for _ in range(2)]
    rope = RopeCache(320, d, lib=luc)
    gen = torch.Generator().manual_seed(3)
    width = (hq + 2 * hkv) * d
    rnd = lambda n: (torch.randn(n, width, generator=gen) * 1.4).to(torch.bfloat16).cuda()  # noqa: E731

    def layer_calls(cache, layer, qkv, out, max_rows):
        q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        cache.append(layer, q, k, v, rope)
        cache.attend(layer, out, q, 320, max_rows)

    for layer_rows in [[rnd(180) for _ in range(layers)]]:
        for c in caches:
            c.extend(i32([100, 15, 65]), rows=180)
            for layer, qkv in enumerate(layer_rows):
                layer_calls(c, layer, qkv.clone(), torch.empty(180, hq * d, dtype=torch.bfloat16, device="cuda"), 100)
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
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    held = [x.clone() for x in qkv_in]
    with torch.cuda.graph(graph):
        for a, b in zip(held, qkv_in):  # (append rotates q in place)
            a.copy_(b)
        step(caches[0], held, outs)
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
        for name in ("lens", "block_tables", "slots", "positions", "start_pos", "state"):
            assert torch.equal(getattr(caches[0].blocks, name), getattr(caches[1].blocks, name)), name
    assert caches[0].blocks.lens.tolist() == [140, 15, 105]
    assert torch.equal(caches[0].k_pool, caches[1].k_pool) and torch.equal(caches[0].v_pool, caches[1].v_pool)
    caches[0].blocks.check()


def test_a_workspace_is_made_before_a_capture(luc):
    cache = Kv4Cache(1, 8, 2, 64, 400, 1, 6000, lib=luc)
    q = torch.zeros(1, 512, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            cache.attend(0, torch.empty_like(q), q, 6000)
    ws = cache.workspace(1, 1, 6000)
    assert cache.workspace(1, 1, 1000) in (None, ws) and not bool(ws.any())


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, "f16"), (12, 2, 128, "bf16")])
def test_maps_and_normed_appends_over_a_16_bit_cache(luc, hq, hkv, d, dtype):
    """DeviceBlocks, qk_norm_rope_append and luc_paged_decode: what a 16-bit loop uses."""
    dt, layers, seqs = DT[dtype], 2, 3
    blocks = DeviceBlocks(30, seqs, 12, 64, lib=luc)
    shape = (30, layers, hkv, PAGE, d)
    kp, vp = (torch.full(shape, float("nan"), dtype=dt, device="cuda") for _ in range(2))
    kp[:], vp[:] = 0, 0
    rope = RopeCache(192, d, lib=luc)
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    norms = [(1 + 0.2 * rnd(d)).to(dt).cuda() for _ in range(2)]
    a, b = hq * d, (hq + hkv) * d
    for new in ([33, 5, 16], [1, 1, 1], [1, 1, 1]):
        total = sum(new)
        blocks.extend(i32(new), rows=total)
        qkv = (rnd(total, b + hkv * d) * 1.4).to(dt).cuda()
        q, k, v = qkv[:, :a], qkv[:, a:b], qkv[:, b:]
        q_out = torch.empty(total, a, dtype=dt, device="cuda")
        luc.qk_norm_rope_append(q, k, v, rope.cos, rope.sin, blocks.positions, blocks.slots, kp, vp, 1, layers, hq, hkv,
                                d, q_norm=norms[0], k_norm=norms[1], q_out=q_out)
    blocks.check()
    ctx = blocks.lens.tolist()
    out = torch.empty_like(q_out)
    luc.paged_decode(out, q_out, kp, vp, blocks.block_tables, blocks.start_pos, seqs, max(ctx), 1, layers, hq, hkv, d,
                     sm_scale(d))
    for s in range(seqs):
        ids = blocks.block_tables[s, :-(-ctx[s] // PAGE)].long()
        kx, vx = (p[ids, 1].double().swapaxes(1, 2).reshape(-1, hkv, d)[:ctx[s]] for p in (kp, vp))
        want, tol = ref.attention(q_out[s:s + 1].double().view(1, hq, d), kx, vx, ctx[s] - 1, sm_scale(d))
        # paged_decode takes P in the cache's type: half a step of it where that is bf16
        tol = tol + (torch.finfo(dt).eps / 2 * vx.abs().amax() if dtype == "bf16" else 0)
        ref.check(out[s:s + 1].view(1, hq, d), want, tol, dt, f"sequence {s} of {ctx[s]}")


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 3, 65]])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128)])
def test_sequences_that_share_pages(luc, hq, hkv, d, rows):
    """A prefix's pages in several tables, as prefix caching leaves them: the same as copies of them."""
    ctx = [700, 300, 1000]
    c = Cache(ctx, hkv, d, seed=9)
    shared = 15                                        # pages of sequence 0 in the other tables too
    for b in (1, 2):
        c.tables[b, :shared] = c.tables[0, :shared]
        c.k[b][:shared * PAGE], c.v[b][:shared * PAGE] = c.k[0][:shared * PAGE], c.v[0][:shared * PAGE]
    c.dev_tables = torch.from_numpy(c.tables).cuda()
    q, out, scale = run(luc, c, rows, hq, "f16")
    verify(c, rows, hq, "f16", q, out, scale)


def test_two_streams_at_once(luc):
    """Steps of two caches on two streams that overlap, with a workspace each: the bits of the same
    steps in turn."""
    hq, hkv, d, steps = 14, 2, 64, 12
    rope = RopeCache(3000, d, lib=luc)
    width = (hq + 2 * hkv) * d

    def prepare(seed):
        gen = torch.Generator().manual_seed(seed)
        cache = Kv4Cache(1, hq, hkv, d, 400, 2, 3000, 2700, lib=luc)
        rnd = lambda n: (torch.randn(n, width, generator=gen) * 1.4).half().cuda()  # noqa: E731
        work = [(i32([1500 + 100 * seed, 900]), rnd(2400 + 100 * seed), 1700)] + [(i32([1, 1]), rnd(2), 1) for _ in range(steps)]
        cache.workspace(2, 1, 3000)
        cache.workspace(2400 + 100 * seed, 1700, 3000)
        return cache, work, [torch.zeros(w.shape[0], hq * d, dtype=torch.float16, device="cuda") for _, w, _ in work]

    def issue(cache, work, outs, i, stream):
        new, qkv, most = work[i]
        cache.extend(new, rows=qkv.shape[0], stream=stream)
        q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        cache.append(0, q, k, v, rope, stream=stream)
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


@pytest.fixture(scope="module")
def model(luc):
    return Qwen2Model(CFG, random_weights(CFG, seed=5, std=0.05), lib=luc, kv_bits=4)


def test_model_attention_is_that_of_its_cache(luc, model):
    """forward() of a prompt, single tokens, a second chunk and a step back: every layer's attention
    against 64 bits over what the cache holds."""
    d, hq = CFG.head_dim, CFG.num_attention_heads
    seen = []
    inner = model.kv.attend

    def attend(layer, out, q, max_ctx, *rest, **kw):
        inner(layer, out, q, max_ctx, *rest, **kw)
        seen.append((layer, out.clone(), q.clone(), max_ctx))

    model.kv.attend = attend
    try:
        rng = np.random.default_rng(2)
        for n, pos in ((40, 0), (1, 40), (1, 41), (70, 42), (2, 30), (1, 32)):
            seen.clear()
            model.forward(rng.integers(0, CFG.vocab_size, n).tolist(), pos)
            assert len(seen) == CFG.num_hidden_layers and int(model.kv.blocks.lens) == pos + n
            ids = model.kv.blocks.block_tables[0, :-(-(pos + n) // PAGE)].cpu().numpy().astype(np.int64)
            for layer, out, q, ctx in seen:
                assert ctx == pos + n
                k, v = (unpack(p, ids, layer, d, x)[0][:ctx] for p, x in ((model.kv.k_pool, False), (model.kv.v_pool, True)))
                want, tol = ref.attention(q.double().view(n, hq, d), k, v, pos, sm_scale(d))
                ref.check(out.view(n, hq, d), want, tol, torch.bfloat16, f"{n} rows at {pos}, layer {layer}")
            assert bool(model.logits().isfinite().all())
    finally:
        del model.kv.attend


def test_model_graph_replays_the_eager_loop(luc, model):
    """capture_decode over a 4-bit cache: the eager loop's tokens, twice from the same prompt (contexts
    below one split: the same arithmetic)."""
    prompt = np.random.default_rng(8).integers(0, CFG.vocab_size, 30).tolist()
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


def test_model_refusals(luc, model):
    w = random_weights(CFG, seed=5)
    with pytest.raises(ValueError, match="kv_bits 8"):
        Qwen2Model(CFG, w, lib=luc, kv_bits=8)
    model.forward([1, 2, 3], 0)
    with pytest.raises(ValueError, match="past the 3 tokens"):
        model.forward([4], 5)
    small = Qwen2Model(CFG, w, num_blocks=2, lib=luc, kv_bits=4)
    with pytest.raises(RuntimeError, match="Out of memory blocks"):
        small.forward(list(range(33)), 0)
    with pytest.raises(RuntimeError, match="Out of memory blocks"):
        small.capture_decode(40)
    small.forward(list(range(32)), 0)
    assert bool(small.logits().isfinite().all())


# ---- attention where its work splits change -------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128)])
def test_many_splits(luc, hq, hkv, d):
    """Contexts of more than 64 and more than 128 splits, beside a short and an empty sequence."""
    c = Cache([70001, 513, 36000, 0], hkv, d, seed=4, layers=1, layer=0)
    rows = [1, 1, 1, 0]
    q, out, scale = run(luc, c, rows, hq, "f16")
    verify(c, rows, hq, "f16", q, out, scale)


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 4), (128, 12, 4)])
def test_longest_first(luc, d, hq, hkv):
    """More workgroups than fit at once, of 64 sequences whose lengths differ in every order, some of them
    empty, past max_ctx or at no position."""
    rng = np.random.default_rng(d)
    ctx = rng.integers(1, 2500, 64)
    ctx[[3, 40]] = 5000
    ctx[[5, 63]] = 1
    rows = [1] * 64
    for b in (0, 17, 18):
        ctx[b], rows[b] = 100, 0
    c = Cache(ctx.tolist(), hkv, d, seed=d, layers=1, layer=0)
    q, out, scale = run(luc, c, rows, hq, "bf16")
    verify(c, rows, hq, "bf16", q, out, scale)
    start = [x - r for x, r in zip(c.ctx, rows)]
    start[7] = -3
    q, got, scale = run(luc, c, rows, hq, "bf16", q=q, max_ctx=3000, start=start)
    at = np.cumsum([0] + rows)
    for b in (3, 7, 40):
        assert bool(got[at[b]].isnan().all())
    verify(c, rows, hq, "bf16", q, got, scale, skip=(3, 7, 40))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,seqs,rows", [
    (8, 1, 64, 3, 2), (8, 1, 64, 3, 6), (8, 1, 64, 3, 7), (8, 1, 64, 2, 16), (8, 1, 64, 2, 17), (3, 3, 64, 3, 48),
    (3, 3, 64, 3, 49), (3, 3, 64, 2, 128), (3, 3, 64, 2, 129), (8, 1, 128, 3, 6), (8, 1, 128, 3, 7), (8, 1, 128, 2, 32),
    (8, 1, 128, 2, 33), (5, 5, 128, 2, 256), (5, 5, 128, 2, 257), (8, 8, 64, 17, 25), (8, 8, 64, 11, 47)])
def test_numbers_of_columns(luc, hq, hkv, d, seqs, rows, dtype):
    """16 and 17, 48 and 49 columns, one workgroup's and one more, tiles above and below the chip's."""
    c = Cache([rows + 37 * b for b in range(seqs)], hkv, d, seed=rows, layers=1, layer=0)
    counts = [rows - (b % 3 if rows > 3 else 0) for b in range(seqs)]
    q, out, scale = run(luc, c, counts, hq, dtype, max_rows=rows, tail=2)
    verify(c, counts, hq, dtype, q, out, scale)
