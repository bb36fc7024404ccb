"""luc_kv4_attention where K, V and the softmax's weights leave the size of a standard normal: V of small and of
mixed sizes, long contexts whose weight is one token's but for a tail, many splits; with bounds without terms
that grow with the context where the kernels' arithmetic has none."""
import math

import numpy as np
import pytest
import torch

import serving_ref as ref
from test_gpu_kv4_attention import DT, PAGE, Cache, run

pytestmark = pytest.mark.gpu
GROUP = ref.GROUP


def cache_of(ks, vs, seed=0):
    """A Cache of sequences with the values ks[b], vs[b] (float32 [ctx, hkv, d]); every other byte 0xff."""
    rng = np.random.default_rng(seed)
    c = object.__new__(Cache)
    c.ctx = [len(x) for x in ks]
    c.hkv, c.d = ks[0].shape[1:]
    c.layers, c.layer = 1, 0
    pages = [-(-n // PAGE) for n in c.ctx]
    c.pages = sum(pages) + 2
    perm = rng.permutation(c.pages).astype(np.int32)
    c.tables = np.full((len(ks), max(pages)), -7, np.int32)
    kp = np.full((c.pages, 1, c.hkv, 10 * c.d), 0xFF, np.uint8)
    vp = kp.copy()
    c.k, c.v = [], []
    at = 0
    for b, n in enumerate(pages):
        ids = perm[at:at + n]
        at += n
        c.tables[b, :n] = ids
        for pool, given, is_v, keep in ((kp, ks[b], False, c.k), (vp, vs[b], True, c.v)):
            x = np.full((n * PAGE, c.hkv, c.d), np.nan, np.float32)
            x[:c.ctx[b]] = given
            slabs, val = ref.pack_pool(np.ascontiguousarray(x.reshape(n, PAGE, c.hkv, c.d).swapaxes(1, 2)), is_v)
            pool[ids, 0] = slabs
            keep.append(torch.from_numpy(np.ascontiguousarray(val.swapaxes(1, 2)).reshape(-1, c.hkv, c.d)[:c.ctx[b]]).cuda())
    c.kp, c.vp = torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda()
    c.dev_tables = torch.from_numpy(c.tables).cuda()
    return c


def bound(q, k, v, start, scale, dtype, few):
    """(out, tolerance without the output's own rounding) of rows q [n, hq, d], all in float64; few: the call has so
    few columns that waves split tokens.

    Weights are held times 2^lift: 12 for few columns, less where V has steps of 1 and more (a weight times a step
    stays below 2^15), and 7 for many.  Of the output:
      sums: f32 sums and products in 16 and 32 steps, each of them relative to the sizes |n s| + |m| of its terms:
        fewer than 64 roundings of 2^-24, and the matrix unit's alignment of subnormals (6 bits), 2^-17 in all
      scores: the same of scale sum |q| (|n s| + |m|), 2^-18 in powers of e
      weights, few columns: bf16 rows have them truncated to fp16 (as has their sum): uniform in 2^-10 of
        themselves.  fp16 rows have two parts.  Either loses up to 2^-24 / 2^lift of the largest, and the product with
        a step two roundings of 2^-25 / 2^lift, times n <= 15
      many columns: V is rounded to fp16, half a step of 2^-11; bf16 rows' K and weights too.  Below 2^-14 weights
        are multiples of 2^-24 / 2^lift
    What is rounded independently for each token is summed as the root of the squares, six times that."""
    n, hq, d = q.shape
    ctx, hkv = k.shape[:2]
    g = hq // hkv
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.empty_like(out)
    at = torch.arange(ctx, device=q.device)

    def groups(x):
        x = x.unflatten(-1, (-1, GROUP))
        return x, x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)

    half, many = 2.0 ** -11, 6 / math.sqrt(3)
    for h in range(hkv):
        (kx, km, _), (vx, vm, vtop) = groups(k[:, h]), groups(v[:, h])
        k_size, v_size = ((x - m + m.abs()).flatten(-2) for x, m in ((kx, km), (vx, vm)))
        step = float((vtop - vm).max()) / 15
        lift = min(12, max(-1, 11 - math.floor(math.log2(max(step, 1e-9))))) if few else 7
        floor = 2.0 ** -lift
        for j in range(h * g, h * g + g):
            for r in range(n):
                x, seen = q[r, j], start + r + 1
                kk, vv = k[:seen, h], v[:seen, h]
                p = torch.softmax(kk @ x * scale, 0)
                o = p @ vv
                away = (vv - o).abs()
                e = abs(scale) * 2.0 ** -18 * (k_size[:seen] @ x.abs()) + 2.0 ** -21
                w2 = torch.zeros_like(p)
                t = 2.0 ** -17 * (p @ v_size[:seen])
                most = p.max() * seen
                if few:
                    if dtype == "bf16":
                        w2 = w2 + 2.0 ** -20 / 12
                    t = t + most * floor * (2.0 ** -24 * vv.abs().max() + 15 * 2.0 ** -24)
                else:
                    t = t + many * half * torch.sqrt((p * p) @ (vv * vv))
                    if dtype == "bf16":
                        w2 = w2 + ((kk * kk) @ (x * x) * (scale * half) ** 2 + half ** 2) / 3
                    t = t + many * p.max() * math.sqrt(seen) * 2.0 ** -25 * floor * vv.abs().max()
                t = t + (p * e) @ away + 6 * torch.sqrt((p * p * w2) @ (away * away))
                out[r, j], tol[r, j] = o, t
    return out, tol


def verify(c, rows, hq, dtype, q, out, scale, few, pick=None):
    r0 = 0
    for b, n in enumerate(rows):
        which = list(range(n)) if pick is None else sorted({x % n for x in pick})
        for r in which:
            row = slice(r0 + r, r0 + r + 1)
            want, tol = bound(q[row].double().view(1, hq, c.d), c.k[b], c.v[b], c.ctx[b] - n + r, scale, dtype, few)
            ref.check(out[row].view(1, hq, c.d), want, tol, DT[dtype], f"sequence {b}, row {r} of {n} at {c.ctx[b]}")
        r0 += n


def normal(rng, ctx, hkv, d, std):
    return rng.standard_normal((ctx, hkv, d), dtype=np.float32) * np.float32(std)


@pytest.mark.parametrize("rows", [1, 3, 60])
@pytest.mark.parametrize("dtype,v_std", [("f16", 1e-2), ("f16", 1e-3), ("f16", 1e-4), ("bf16", 1e-3), ("bf16", 1e-5),
                                         ("f16", 1.0), ("bf16", 40.0), ("f16", 1000.0)])
@pytest.mark.parametrize("hq,hkv,d", [(10, 2, 64), (5, 1, 128)])
def test_sizes_of_v(luc, hq, hkv, d, dtype, v_std, rows):
    rng = np.random.default_rng(rows)
    ctx = [300, 1100]
    c = cache_of([normal(rng, n, hkv, d, 1.4) for n in ctx], [normal(rng, n, hkv, d, v_std) for n in ctx])
    q, out, scale = run(luc, c, [rows, rows], hq, dtype)
    verify(c, [rows, rows], hq, dtype, q, out, scale, rows < 10, pick=(0, 1, -1))


@pytest.mark.parametrize("rows", [1, 2, 40])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_sizes_of_v_along_a_context(luc, d, dtype, rows):
    """V of 0.01 at first, then of 1, 30 and 2000, then of 0.01 again; and in the other order."""
    rng = np.random.default_rng(d)
    sizes = np.repeat(np.float32([0.01, 1.0, 30.0, 2000.0, 0.01]), [130, 200, 37, 16, 217])[:, None, None]
    ks = [normal(rng, 600, 2, d, 1.4) for _ in range(2)]
    vs = [normal(rng, 600, 2, d, 1.0) * s for s in (sizes, sizes[::-1])]
    c = cache_of(ks, vs)
    q, out, scale = run(luc, c, [rows, rows], 6, dtype)
    verify(c, [rows, rows], 6, dtype, q, out, scale, rows < 10, pick=(0, -1))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx,v_mean,v_std", [(30000, 1.0, 0.2), (30, 1000.0, 0.5)])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (5, 1, 128)])
def test_one_token_and_a_tail(luc, hq, hkv, d, ctx, v_mean, v_std, dtype, rows):
    """Position 0 has nearly all the weight and V = 0; the others have 2^-25.5 of it each, and the output is theirs."""
    rng = np.random.default_rng(d)
    rows = min(rows, ctx - 5)
    k, v = normal(rng, ctx, hkv, d, 0.05), normal(rng, ctx, hkv, d, v_std) + np.float32(v_mean)
    scale = d ** -0.5
    k[0] = 25.5 * math.log(2) / (scale * d)   # q is near 1 throughout
    v[0] = 0
    c = cache_of([k], [v])
    gen = torch.Generator().manual_seed(2)
    q = (1 + 0.02 * torch.randn(rows, hq * d, generator=gen)).to(DT[dtype]).cuda()
    q, out, scale = run(luc, c, [rows], hq, dtype, q=q, scale=scale)
    assert 2e-4 < float(out.double().mean()) < 2e-3
    verify(c, [rows], hq, dtype, q, out, scale, rows < 10, pick=(0, 1, -1))


def splits(luc, batch, total, max_rows, max_ctx, hq, hkv, d):
    """Splits of a call with few columns, from its workspace: [counters][(m, l), o] of 8 columns a tile."""
    tiles = -(-min(total, max_rows) * (hq // hkv) // 8)
    size = luc.lib.luc_kv4_workspace_size(batch, total, max_rows, max_ctx, hq, hkv, d)
    return max(0, size - (1 << 18)) // (batch * hkv * tiles * 8 * (8 + 4 * d))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx,least", [(33001, 65), (70001, 129), (131072, 256)])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (3, 1, 128)])
def test_one_sequence_of_many_splits(luc, hq, hkv, d, ctx, least, dtype):
    """More than 64 and more than 128 splits, and as many as there may be, merged by one workgroup, within a
    bound that an output without one split's 512 tokens passes."""
    rng = np.random.default_rng(ctx)
    assert splits(luc, 1, 1, 1, ctx, hq, hkv, d) >= least
    v = normal(rng, ctx, hkv, d, 1.0)
    v += np.float32(3) * np.sin(np.arange(ctx, dtype=np.float32) * 0.01)[:, None, None]  # every split's part differs
    c = cache_of([normal(rng, ctx, hkv, d, 0.5)], [v])
    for rows in ([1], [2]):
        q, out, scale = run(luc, c, rows, hq, dtype)
        verify(c, rows, hq, dtype, q, out, scale, True)
        want, tol = bound(q[:1].double().view(1, hq, d), c.k[0], c.v[0], ctx - rows[0], scale, dtype, True)
        half = torch.finfo(DT[dtype]).eps / 2
        # leaving 512 tokens near the start out
        x = q[0].double().view(hq, d)
        for j in range(hq):
            p = torch.softmax(c.k[0][:ctx - rows[0] + 1, j // (hq // hkv)] @ x[j] * scale, 0)
            p[512:1024] = 0
            less = p @ c.v[0][:len(p), j // (hq // hkv)] / p.sum()
            far = (less - want[0, j]).abs() / (tol[0, j] + half * want[0, j].abs())
            assert float(far.max()) > 3


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx", [[1, 40], [500, 3, 1000, 77], [5000], [2049, 700]], ids=lambda c: "_".join(map(str, c)))
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128), (8, 8, 64), (28, 4, 128)])
def test_a_bound_far_above_every_context(luc, hq, hkv, d, ctx, dtype):
    """max_ctx as a captured step has it: launches with more splits than any context, for one row a sequence and for
    several."""
    rng = np.random.default_rng(len(ctx))
    c = cache_of([normal(rng, n, hkv, d, 1.4) for n in ctx], [normal(rng, n, hkv, d, 1.0) for n in ctx])
    wide = torch.full((len(ctx), 2500), -7, dtype=torch.int32, device="cuda")
    wide[:, :c.tables.shape[1]] = c.dev_tables
    for rows in (1, 2, 30):
        counts = [min(rows, n) for n in ctx]
        need = [luc.lib.luc_kv4_workspace_size(len(ctx), sum(counts), max(counts), m, hq, hkv, d)
                for m in (max(ctx), 40000)]
        assert need[1] > need[0]
        q, out, scale = run(luc, c, counts, hq, dtype, max_ctx=40000, tables=wide)
        units = len(ctx) * hkv * -(-max(counts) * (hq // hkv) // 8)
        cols = max(counts) * (hq // hkv)
        verify(c, counts, hq, dtype, q, out, scale, cols <= 16 or (cols <= 48 and units <= 512), pick=(0, -1))


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (5, 1, 128)])
def test_keys_far_from_zero(luc, hq, hkv, d, dtype, rows):
    """A group of K at 1000 cos(t) + N(0, 1.4), which q's own group, of mean 0, takes out of the scores: few columns
    multiply m by the sum of q, which has to be as exact as q.

    q is a multiple of 2^-14 (2^-6 in bf16) below 8, so 32 of it are summed exactly.  A score's error: roundings of
    2^-24 of sum n s q and m sum q by group, fewer than 4; and in n q, whose products the matrix unit aligns by
    fp16's smallest exponent, 2^-23 where q's largest is in [2^14, 2^15) and n is 2^-24 n, spread evenly."""
    ctx = [300, 1000]
    rng = np.random.default_rng(5)
    ks = [normal(rng, n, hkv, d, 1.4) for n in ctx]
    for k in ks:
        k[:, :, 32:64] += 1000 * np.cos(np.arange(len(k), dtype=np.float32))[:, None, None]
    c = cache_of(ks, [normal(rng, n, hkv, d, 1.0) for n in ctx])
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2 * rows, hq, d, generator=gen) * 1.4
    x[:, :, 32:64] -= x[:, :, 32:64].mean(-1, keepdim=True)
    fine = 2.0 ** (14 if dtype == "f16" else 6)
    q = ((x * fine).round() / fine).reshape(2 * rows, hq * d).to(DT[dtype]).cuda()
    if dtype == "bf16":  # (its rounding leaves a sum, which the last element takes)
        y = q.view(2 * rows, hq, d)[:, :, 32:64].float()
        y = (y * 8).round() / 8
        y[..., 31] -= y.sum(-1)
        q.view(2 * rows, hq, d)[:, :, 32:64] = y.to(q.dtype)
    q, out, scale = run(luc, c, [rows, rows], hq, dtype, q=q)
    for row in range(2 * rows):
        b, seen = row // rows, ctx[row // rows] - rows + row % rows + 1
        want = torch.empty((1, hq, d), dtype=torch.float64, device="cuda")
        tol = torch.empty_like(want)
        for j in range(hq):
            qj = q[row].double().view(hq, d)[j]
            k, v = (t[:seen, j // (hq // hkv)] for t in (c.k[b], c.v[b]))
            kg = k.unflatten(-1, (-1, GROUP))
            m = kg.amin(-1)
            qg = qj.view(-1, GROUP)
            ns = ((kg - m[..., None]) * qg).sum(-1).abs().sum(-1) + (m * qg.sum(-1)).abs().sum(-1)
            step = (kg.amax(-1) - m).amax(-1) / 15
            unit = 2.0 ** (math.floor(math.log2(float(qj.abs().max()))) - 13)
            p = torch.softmax(k @ qj * scale, 0)
            o = p @ v
            away = (v - o).abs()
            e = scale * 2.0 ** -22 * ns + 2.0 ** -21
            w2 = (scale * step * unit) ** 2 * d / 12 + (2.0 ** -20 / 12 if dtype == "bf16" else 0)
            want[0, j] = o
            tol[0, j] = (p * e) @ away + 6 * torch.sqrt((p * p * w2) @ (away * away)) + \
                2.0 ** -17 * (p @ (v.abs() + 2 * v.abs().amax(-1, keepdim=True)))
        ref.check(out[row].view(1, hq, d), want, tol, DT[dtype], f"row {row}, {seen} tokens")


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("top", [2.0 ** 19, 2.0 ** 22, 2.0 ** 25, 2.0 ** 28])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (5, 1, 128)])
def test_scores_whose_roundings_are_powers_of_two(luc, hq, hkv, d, top, dtype, rows):
    """Scores up to 2^26 (many columns 2^28), where a step of 32 bits is some powers of e: the largest one's V is the output, where the next lies
    2^-8 of it behind (K in fp16, 2^-11 of each product, moves a score of many terms less)."""
    rng = np.random.default_rng(7)
    ctx = 900
    top = top if rows == 40 else min(top, 2.0 ** 26)
    k = normal(rng, ctx, hkv, d, 300.0) * (1 + np.arange(ctx, dtype=np.float32) / 300)[:, None, None]
    c = cache_of([k], [normal(rng, ctx, hkv, d, 1.0)])
    gen = torch.Generator().manual_seed(4)
    q = (torch.randn(rows, hq * d, generator=gen) * 50).to(DT[dtype]).cuda()
    hidden = torch.arange(ctx, device="cuda")[None] > ctx - rows + torch.arange(rows, device="cuda")[:, None]
    score = torch.stack([(q.double().view(rows, hq, d)[:, j] @ c.k[0][:, j // (hq // hkv)].t().contiguous())
                         .masked_fill(hidden, -math.inf) for j in range(hq)], 1)
    scale = top / float(score.max())
    q, out, _ = run(luc, c, [rows], hq, dtype, q=q, scale=scale)
    best = score.topk(2, -1)
    sure = best.values[..., 0] - best.values[..., 1] > 2.0 ** -8 * best.values[..., 0]
    assert float(sure.double().mean()) > 0.8 and float(best.values.min()) * scale > top / 8
    want = torch.stack([c.v[0][best.indices[:, j, 0], j // (hq // hkv)] for j in range(hq)], 1)
    got = out.view(rows, hq, d)
    assert bool(got.isfinite().all())
    # V in fp16 (many columns) and the output's rounding
    tol = (2.0 ** -11 + torch.finfo(DT[dtype]).eps / 2) * want.abs() * 1.01 + 2.0 ** -20
    assert bool(((got.double() - want).abs() <= tol)[sure].all())
