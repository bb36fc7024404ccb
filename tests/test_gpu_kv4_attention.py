"""luc_kv4_attention against 64-bit attention over the values that the 4-bit cache holds."""
import numpy as np
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


class Cache:
    """4-bit pools whose sequences have `ctx` tokens on shuffled pages; every other byte, the
    tokens behind a context and the pages of nobody, is 0xff: n = 15, s = m = NaN."""

    def __init__(self, ctx, hkv, d, seed=0, layers=2, layer=1, k_std=1.4, v_std=1.0, spare=3):
        rng = np.random.default_rng(seed)
        self.ctx, self.hkv, self.d, self.layers, self.layer = ctx, hkv, d, layers, layer
        pages = [-(-c // PAGE) for c in ctx]
        self.pages = sum(pages) + spare
        perm = rng.permutation(self.pages).astype(np.int32)
        stride = max(pages + [1])
        self.tables = np.full((len(ctx), stride), -7, np.int32)
        kp = np.full((self.pages, layers, hkv, 10 * d), 0xFF, np.uint8)
        vp = kp.copy()
        self.k, self.v = [], []
        at = 0
        for b, (c, n) in enumerate(zip(ctx, pages)):
            ids = perm[at:at + n]
            at += n
            self.tables[b, :n] = ids
            for pool, std, is_v, keep in ((kp, k_std, False, self.k), (vp, v_std, True, self.v)):
                x = np.full((n * PAGE, hkv, d), np.nan, np.float32)
                x[:c] = rng.standard_normal((c, hkv, d), dtype=np.float32) * std
                slabs, val = ref.pack_pool(np.ascontiguousarray(x.reshape(n, PAGE, hkv, d).swapaxes(1, 2)), is_v)
                pool[ids, layer] = slabs
                keep.append(torch.from_numpy(np.ascontiguousarray(val.swapaxes(1, 2)).reshape(-1, hkv, d)[:c]).cuda())
        self.kp, self.vp = torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda()
        self.dev_tables = torch.from_numpy(self.tables).cuda()


def run(luc, c, rows, hq, dtype, seed=1, max_ctx=None, max_rows=None, packed=True, tail=0, q_std=1.4, scale=None,
        q=None, q_extra=0, out_extra=0, ws=None, stream=None, start=None, tables=None, num_blocks=None):
    """Rows of every sequence at the end of its context: (q, out, scale)."""
    dt, n = DT[dtype], len(c.ctx)
    total = sum(rows) + tail
    gen = torch.Generator().manual_seed(seed)
    if q is None:
        q = (torch.randn(total, hq * c.d + q_extra, generator=gen) * q_std).to(dt).cuda()[:, :hq * c.d]
    out = torch.full((total, hq * c.d + out_extra), 7.0, dtype=dt, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda") if packed else None
    if start is None:
        start = [x - r for x, r in zip(c.ctx, rows)]
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    max_ctx = max_ctx or max(c.ctx + [1])
    max_rows = max_rows or max(rows + [1])
    scale = scale if scale is not None else c.d ** -0.5
    if ws is None:
        ws = luc.kv4_workspace(n, total, max_rows, max_ctx, hq, c.hkv, c.d)
    print(f"  attention: ctx {c.ctx[:8]} rows {rows[:8]} heads {hq}/{c.hkv}x{c.d} {dtype} max_ctx {max_ctx} "
          f"max_rows {max_rows} workspace {0 if ws is None else ws.numel() * 4}", flush=True)
    luc.kv4_attention(out[:, :hq * c.d], q, c.kp, c.vp, c.dev_tables if tables is None else tables, st, n, total,
                      max_rows, max_ctx, c.layer, c.layers, hq, c.hkv, c.d, scale, cu_seqlens=cu, workspace=ws,
                      stream=stream, num_blocks=num_blocks)
    torch.cuda.synchronize()
    if ws is not None:
        assert not ws[:1024].any(), "arrival counters"
    assert bool((out[:, hq * c.d:] == 7).all()), "columns behind a row"
    assert bool((out[sum(rows):] == 7).all()), "rows behind the last sequence"
    return q, out[:, :hq * c.d], scale


def verify(c, rows, hq, dtype, q, out, scale, skip=()):
    r0 = 0
    for b, n in enumerate(rows):
        if n and b not in skip:
            want, tol = ref.attention(q[r0:r0 + n].double().view(n, hq, c.d), c.k[b], c.v[b], c.ctx[b] - n, scale)
            ref.check(out[r0:r0 + n].view(n, hq, c.d), want, tol, DT[dtype], f"sequence {b}, {n} rows of {c.ctx[b]}")
        r0 += n


HEADS = [(14, 2, 64), (12, 2, 128), (8, 8, 64), (16, 2, 128), (5, 1, 128), (4, 2, 64), (3, 1, 64), (28, 4, 128)]
CONTEXTS = [[1], [15, 16, 17], [31, 32, 33, 1], [127, 128, 129, 64], [500, 3, 1000, 77], [5000]]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx", CONTEXTS, ids=lambda c: "_".join(map(str, c)))
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_against_64_bit_attention(luc, hq, hkv, d, ctx, dtype):
    c = Cache(ctx, hkv, d, seed=len(ctx))
    rows = [1] * len(ctx)
    q, out, scale = run(luc, c, rows, hq, dtype, packed=False)
    verify(c, rows, hq, dtype, q, out, scale)
    # packed rows are the same; a looser bound plans other splits
    q2, out2, _ = run(luc, c, rows, hq, dtype, q=q, max_ctx=len(c.tables[0]) * PAGE)
    verify(c, rows, hq, dtype, q2, out2, scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx,rows", [
    ([2, 40], [2, 2]), ([3], [3]), ([33, 70, 5], [5, 0, 5]), ([64, 200], [20, 33]), ([100], [100]),
    ([300, 17, 1, 640], [300, 17, 1, 40]), ([2100], [130]), ([257, 1000], [256, 257]), ([9000], [70])],
    ids=lambda x: "_".join(map(str, x)))
@pytest.mark.parametrize("hq,hkv,d", HEADS[:5])
def test_rows_against_64_bit_attention(luc, hq, hkv, d, ctx, rows, dtype):
    c = Cache(ctx, hkv, d, seed=sum(rows))
    q, out, scale = run(luc, c, rows, hq, dtype, tail=3, q_extra=8, out_extra=4)
    verify(c, rows, hq, dtype, q, out, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [90, 33]])
def test_scales_and_large_scores(luc, d, rows):
    """Scores of both signs far from 0, growing along the context (the running maximum moves),
    a negative scale, and a query of zeros."""
    c = Cache([700, 650], 2, d, seed=3, k_std=4.0)
    for scale, std in ((0.5, 4.0), (-0.25, 4.0), (1.0, 0.0), (3e-3, 200.0)):
        q, out, _ = run(luc, c, rows, 6, "f16", q_std=std, scale=scale)
        verify(c, rows, 6, "f16", q, out, scale)


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 40, 40]])
@pytest.mark.parametrize("dtype", ["bf16"])
def test_queries_outside_fp16(luc, rows, dtype):
    """bf16 queries of 1e-30 and 1e30: products in range after their scale."""
    c = Cache([100, 600, 333], 2, 128, seed=8)
    for std, scale in ((1e-30, 1e29), (1e30, 1e-31)):
        q, out, _ = run(luc, c, rows, 8, dtype, q_std=std, scale=scale)
        verify(c, rows, 8, dtype, q, out, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [[1], [2], [24], [200]])
def test_what_lies_behind_a_position_stays_there(luc, d, rows):
    """NaN K and V at some of the new rows' own tokens: a row sees those at and before its position only."""
    n, ctx = rows[0], 420
    c = Cache([ctx], 2, d, seed=12)
    start = ctx - n
    q, clean, scale = run(luc, c, rows, 8, "f16")
    verify(c, rows, 8, "f16", q, clean, scale)
    # V: group 1 of head 0 is NaN at token t; K: head 1 is NaN at token u
    t, u = start + n // 2, start + n // 3
    page, off = int(c.tables[0, t // PAGE]), t % PAGE
    nan = torch.tensor([0x7E00], dtype=torch.int16).view(torch.float16).cuda()
    vsm = c.vp[page, 1, 0, 8 * d:].view(torch.float16).view(2, d // 32, 2, 8)
    vsm[off // 8, 1, :, off % 8] = nan
    page, off = int(c.tables[0, u // PAGE]), u % PAGE
    c.kp[page, 1, 1, 8 * d:].view(torch.float16).view(16, d // 32, 2)[off, 0] = nan
    _, out, _ = run(luc, c, rows, 8, "f16", q=q)
    o, w = out.view(n, 8, d), clean.view(n, 8, d)
    assert torch.equal(o[:t - start, :4], w[:t - start, :4])
    assert bool(o[t - start:, :4, 32:64].isnan().all())
    rest = [x for x in range(d) if not 32 <= x < 64]
    assert torch.equal(o[t - start:, :4, rest], w[t - start:, :4, rest])
    assert torch.equal(o[:u - start, 4:], w[:u - start, 4:])
    assert bool(o[u - start:, 4:].isnan().all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [2, 3, 1, 4], [60, 70, 1, 50]])
def test_contexts_out_of_bounds_are_nan(luc, d, rows):
    """Contexts past max_ctx, negative positions, more rows than max_rows, pages outside the pool."""
    c = Cache([300, 200, 150, 400], 2, d, seed=5)
    hq = 10
    q, clean, scale = run(luc, c, rows, hq, "bf16")
    verify(c, rows, hq, "bf16", q, clean, scale)
    ends = np.cumsum(rows)
    seq = [slice(e - r, e) for e, r in zip(ends, rows)]
    _, out, _ = run(luc, c, rows, hq, "bf16", q=q, max_ctx=350)
    assert bool(out[seq[3]].isnan().all()) and bool(out[:ends[2]].isfinite().all())
    start = [x - r for x, r in zip(c.ctx, rows)]
    _, out, _ = run(luc, c, rows, hq, "bf16", q=q, start=[start[0], -1, start[2], -(1 << 31)])
    assert bool(out[seq[1]].isnan().all()) and bool(out[seq[3]].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(1, 3))
    if max(rows) > 1:
        most = sorted(rows)[-2]
        _, out, _ = run(luc, c, rows, hq, "bf16", q=q, max_rows=most)
        big = rows.index(max(rows))
        assert bool(out[seq[big]].isnan().all())
        verify(c, rows, hq, "bf16", q, out, scale, skip=(big,))
    # a bad page at position 96 of sequence 0 and at 384 of sequence 3 (its last)
    tables = c.dev_tables.clone()
    tables[0, 6] = -1
    tables[3, 24] = c.pages
    _, out, _ = run(luc, c, rows, hq, "bf16", q=q, tables=tables)
    assert bool(out[seq[0]].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(0, 3))
    first = max(0, 384 - (400 - rows[3]))
    assert bool(out[seq[3]][first:].isnan().all())
    assert torch.equal(out[seq[3]][:first], clean[seq[3]][:first])
    # a pool of fewer pages than the tables name
    _, out, _ = run(luc, c, rows, hq, "bf16", q=q, num_blocks=int(c.tables[2, :10].max()))
    assert bool(out[seq[2]].isnan().all())


def test_one_workspace_for_calls_of_other_sizes(luc):
    """Decode and prompt calls of several sizes in turn on one workspace, and again."""
    calls = [(Cache([3000, 1000], 2, 128, seed=1), [1, 1], 12), (Cache([600], 2, 64, seed=2), [300], 14),
             (Cache([5000], 1, 64, seed=3), [1], 8), (Cache([2000, 30], 2, 128, seed=4), [100, 30], 16)]
    need = max(luc.lib.luc_kv4_workspace_size(len(c.ctx), sum(r), max(r), max(c.ctx), hq, c.hkv, c.d)
               for c, r, hq in calls)
    ws = torch.zeros(need // 4, dtype=torch.float32, device="cuda")
    first = [run(luc, c, r, hq, "f16", ws=ws)[1] for c, r, hq in calls]
    for (c, r, hq), was in zip(reversed(calls), reversed(first)):
        q, out, scale = run(luc, c, r, hq, "f16", ws=ws)
        assert torch.equal(out, was)
        verify(c, r, hq, "f16", q, out, scale)


@pytest.mark.parametrize("rows", [[1, 1, 1], [50, 70, 1]])
def test_another_stream_and_a_captured_call(luc, rows):
    c = Cache([900, 1500, 200], 2, 128, seed=7)
    q, want, scale = run(luc, c, rows, 12, "bf16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert torch.equal(run(luc, c, rows, 12, "bf16", q=q, stream=stream)[1], want)
    total = sum(rows)
    ws = luc.kv4_workspace(3, total, max(rows), 1500, 12, 2, 128)
    out = torch.zeros((total, 12 * 128), dtype=q.dtype, device="cuda")
    q_in = q.clone().contiguous()
    st = torch.tensor([x - r for x, r in zip(c.ctx, rows)], dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        luc.kv4_attention(out, q_in, c.kp, c.vp, c.dev_tables, st, 3, total, max(rows), 1500, 1, 2, 12, 2, 128, scale,
                          cu_seqlens=cu, workspace=ws)
    for seed in range(4):
        q_in.copy_((torch.randn(q_in.shape, generator=torch.Generator().manual_seed(seed)) * 1.4).to(q.dtype))
        graph.replay()
        eager = run(luc, c, rows, 12, "bf16", q=q_in)[1]
        assert torch.equal(out, eager)


def test_offsets_past_32_bits(luc):
    """A sequence on the last pages of pools of more than 4 GiB."""
    c = Cache([200, 90], 4, 128, seed=6, layers=1, layer=0)
    q, want, scale = run(luc, c, [1, 60], 8, "f16")
    verify(c, [1, 60], 8, "f16", q, want, scale)
    more = (1 << 32) // (4 * 1280) + 7
    kp = torch.zeros((more + c.pages, 1, 4, 1280), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    kp[more:], vp[more:] = c.kp, c.vp
    c.kp, c.vp, c.pages = kp, vp, more + c.pages
    tables = torch.where(c.dev_tables >= 0, c.dev_tables + more, c.dev_tables)
    assert torch.equal(run(luc, c, [1, 60], 8, "f16", q=q, tables=tables)[1], want)
