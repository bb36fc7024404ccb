"""luc_kv8_attention, luc_kv8_select and luc_kv8_sparse_attention against 64-bit results over the values that the
8-bit cache holds."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
import serving_ref

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


class Cache:
    """8-bit pools whose sequences have `ctx` tokens on shuffled pages; every other byte, the tokens behind
    a context and the pages of nobody, is NaN, and so are the scales of nobody's pages.  spread: powers of two
    by which the pages' sizes differ."""

    def __init__(self, ctx, hkv, d, seed=0, layers=2, layer=1, k_std=1.4, v_std=1.0, spare=3, spread=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.hkv, self.d, self.layers, self.layer = ctx, hkv, d, layers, layer
        counts = [-(-c // PAGE) for c in ctx]
        self.pages = sum(counts) + spare
        perm = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((len(ctx), max(counts + [1])), -7, np.int32)
        kp = np.full((self.pages, layers, hkv, 16 * d), 0xFF, np.uint8)
        vp = np.full_like(kp, 0x7F)
        self.scales = np.full((self.pages, layers, hkv, 2), np.nan, np.float32)
        self.bounds = np.zeros((self.pages, layers, hkv, 2, d), np.uint8)
        self.k, self.v = [], []
        at = 0
        for b, (c, n) in enumerate(zip(ctx, counts)):
            ids = perm[at:at + n]
            at += n
            self.tables[b, :n] = ids
            for is_v, (pool, std, keep) in enumerate(((kp, k_std, self.k), (vp, v_std, self.v))):
                x = rng.standard_normal((n * PAGE, hkv, d)) * std
                x[c:] = np.nan
                x = x.reshape(n, PAGE, hkv, d).swapaxes(1, 2)
                if spread:
                    x = x * 2.0 ** rng.integers(-spread, spread + 1, (n, hkv, 1, 1))
                scale = 2.0 ** ref.exponents(np.nanmax(np.abs(x), (2, 3))) if n else np.empty((0, hkv))
                codes = ref.encode(x / scale[..., None, None])
                if not is_v and n:
                    y = np.where(np.isnan(x), np.nan, ref.TABLE[codes])
                    self.bounds[ids, layer] = ref.encode(np.stack([np.nanmax(y, 2), np.nanmin(y, 2)], 2))
                pool[ids, layer] = (codes.reshape(n, hkv, 4, 4, d).swapaxes(-1, -2) if is_v else codes).reshape(n, hkv, 16 * d)
                self.scales[ids, layer, :, is_v] = scale
                val = ref.TABLE[codes] * scale[..., None, None]
                keep.append(torch.from_numpy(np.ascontiguousarray(val.swapaxes(1, 2)).reshape(-1, hkv, d)[:c]).cuda())
        self.kp, self.vp, self.sp = (torch.from_numpy(x).cuda() for x in (kp, vp, self.scales))
        self.bp = torch.from_numpy(self.bounds).cuda()
        self.dev_tables = torch.from_numpy(self.tables).cuda()


def make_q(c, total, hq, dtype, seed=1, std=1.4, extra=0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(total, hq * c.d + extra, generator=gen) * std).to(DT[dtype]).cuda()[:, :hq * c.d]


def run(luc, c, rows, hq, dtype, seed=1, max_ctx=None, max_rows=None, packed=True, tail=0, q_std=1.4, scale=None,
        q=None, q_extra=0, out_extra=0, ws=None, stream=None, start=None, tables=None, num_blocks=None, columns=False):
    """Rows of every sequence at the end of its context: (q, out, scale).  columns: sizes of a call that allows for
    so many rows that it goes to the kernel for prompts, whatever rows there are."""
    n = len(c.ctx)
    if columns:
        tail = max(tail, 12000 // (n * hq))
        max_rows = max_rows or sum(rows) + tail
        q = q if q is None or len(q) == sum(rows) + tail else torch.cat([q, q[:1].expand(tail, -1)])
    total = sum(rows) + tail
    q = make_q(c, total, hq, dtype, seed, q_std, q_extra) if q is None else q
    out = torch.full((total, hq * c.d + out_extra), 7.0, dtype=DT[dtype], device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda") if packed else None
    start = [x - r for x, r in zip(c.ctx, rows)] if start is None else start
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    max_ctx, max_rows = max_ctx or max(c.ctx + [1]), max_rows or max(rows + [1])
    scale = scale if scale is not None else c.d ** -0.5
    ws = luc.kv8_workspace(n, total, max_rows, max_ctx, hq, c.hkv, c.d) if ws is None else ws
    print(f"  attention8: ctx {c.ctx[:8]} rows {rows[:8]} heads {hq}/{c.hkv}x{c.d} {dtype} max_ctx {max_ctx} "
          f"max_rows {max_rows} workspace {0 if ws is None else ws.numel() * 4}", flush=True)
    luc.kv8_attention(out[:, :hq * c.d], q, c.kp, c.vp, c.sp, c.dev_tables if tables is None else tables, st, n, total,
                      max_rows, max_ctx, c.layer, c.layers, hq, c.hkv, c.d, scale, cu_seqlens=cu, workspace=ws,
                      stream=stream, num_blocks=num_blocks)
    torch.cuda.synchronize()
    if ws is not None:
        assert not ws[:65536].any(), "arrival counters"
    assert bool((out[:, hq * c.d:] == 7).all()), "columns behind a row"
    assert bool((out[sum(rows):] == 7).all()), "rows behind the last sequence"
    return q, out[:, :hq * c.d], scale


def verify(c, rows, hq, dtype, q, out, scale, skip=()):
    r0 = 0
    for b, n in enumerate(rows):
        if n and b not in skip:
            pos = torch.arange(c.ctx[b], device="cuda")
            seen = pos[None] <= (c.ctx[b] - n + torch.arange(n, device="cuda"))[:, None]
            want, tol = ref.attention(q[r0:r0 + n].double().view(n, hq, c.d), c.k[b], c.v[b], seen, scale, DT[dtype])
            serving_ref.check(out[r0:r0 + n].view(n, hq, c.d), want, tol, DT[dtype], f"sequence {b}, {n} rows of {c.ctx[b]}")
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
    q, out, scale = run(luc, c, rows, hq, dtype, q_extra=8, out_extra=4, columns=True)
    verify(c, rows, hq, dtype, q, out, scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx,rows", [([4100], [230]), ([6000, 3500, 40], [100, 90, 1]), ([1100, 5000], [2, 200])],
                         ids=lambda x: "_".join(map(str, x)))
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_rows_over_long_contexts(luc, hq, hkv, d, ctx, rows, dtype):
    """Prompts' rows whose contexts are split."""
    c = Cache(ctx, hkv, d, seed=sum(rows))
    q, out, scale = run(luc, c, rows, hq, dtype, tail=1)
    verify(c, rows, hq, dtype, q, out, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [90, 33]])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("columns", [False, True])
def test_scales_and_large_scores(luc, d, rows, dtype, columns):
    """Scores of both signs far from 0 (the running maximum moves), a negative scale, a query of zeros, and
    pages whose sizes differ by up to 2^20."""
    c = Cache([700, 650], 2, d, seed=3, k_std=4.0)
    for scale, std in ((0.5, 4.0), (-0.25, 4.0), (1.0, 0.0), (3e-3, 200.0), (0.0, 1.0)):
        q, out, _ = run(luc, c, rows, 6, dtype, q_std=std, scale=scale, columns=columns)
        verify(c, rows, 6, dtype, q, out, scale)
    c = Cache([700, 650], 2, d, seed=4, k_std=0.02, v_std=1.0, spread=5)
    q, out, scale = run(luc, c, rows, 6, dtype, columns=columns)
    verify(c, rows, 6, dtype, q, out, scale)
    c = Cache([300, 150], 2, d, seed=5, v_std=2.0 ** -9)  # values near fp16's subnormals
    q, out, scale = run(luc, c, rows, 6, dtype, columns=columns)
    verify(c, rows, 6, dtype, q, out, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ctx,n,columns", [(40, 1, False), (40, 3, False), (200, 70, False), (40, 3, True), (200, 70, True)])
def test_values_that_are_not_numbers(luc, d, ctx, n, dtype, columns):
    """A NaN of V reaches its dimension of the rows that see its token, and nothing else; one of K the whole
    row's head.  Rows before it are as if it were not there."""
    hq = 8
    start = ctx - n
    t = start + n // 2          # between the rows' limits (the row's own token, for one)
    c = Cache([ctx], 2, d, seed=7)
    q, clean, scale = run(luc, c, [n], hq, dtype, columns=columns)
    page, off = int(c.tables[0, t // PAGE]), t % PAGE
    dim = 37
    c.vp[page, c.layer, 0, (off // 4 * d + dim) * 4 + off % 4] = 0xFF
    u = start + n - 1           # the last row's own
    c.kp[int(c.tables[0, u // PAGE]), c.layer, 1, (u % PAGE) * d + 5] = 0x7F
    _, out, _ = run(luc, c, [n], hq, dtype, q=q, columns=columns)
    o, w = out[:n].view(n, hq, d), clean[:n].view(n, hq, d)
    rest = [x for x in range(d) if x != dim]
    assert torch.equal(o[:, :4, rest], w[:, :4, rest])
    assert torch.equal(o[:t - start, :4], w[:t - start, :4])
    assert bool(o[t - start:, :4, dim].isnan().all())
    assert torch.equal(o[:u - start, 4:], w[:u - start, 4:])
    assert bool(o[u - start:, 4:].isnan().all())
    # far before every limit, too
    page = int(c.tables[0, 0])
    c.vp[page, c.layer, 1, (0 * d + 11) * 4 + 2] = 0x7F
    if n < 10:
        _, out, _ = run(luc, c, [n], hq, dtype, q=q, columns=columns)
        assert bool(out[:n].view(n, hq, d)[:, 4:, 11].isnan().all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,columns", [([1, 1, 1, 1], False), ([2, 3, 1, 4], False), ([60, 70, 1, 50], False),
                                          ([2, 3, 1, 4], True), ([60, 70, 1, 50], True)])
def test_contexts_out_of_bounds_are_nan(luc, d, rows, columns):
    """Contexts past max_ctx, negative positions, more rows than max_rows, pages outside the pool."""
    c = Cache([300, 200, 150, 400], 2, d, seed=5)
    hq = 10
    q, clean, scale = run(luc, c, rows, hq, "bf16", columns=columns)
    verify(c, rows, hq, "bf16", q, clean, scale)
    ends = np.cumsum(rows)
    seq = [slice(e - r, e) for e, r in zip(ends, rows)]
    _, out, _ = run(luc, c, rows, hq, "bf16", columns=columns, q=q, max_ctx=350)
    assert bool(out[seq[3]].isnan().all()) and bool(out[:ends[2]].isfinite().all())
    start = [x - r for x, r in zip(c.ctx, rows)]
    _, out, _ = run(luc, c, rows, hq, "bf16", columns=columns, q=q, start=[start[0], -1, start[2], -(1 << 31)])
    assert bool(out[seq[1]].isnan().all()) and bool(out[seq[3]].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(1, 3))
    if max(rows) > 1:
        most = sorted(rows)[-2]
        _, out, _ = run(luc, c, rows, hq, "bf16", columns=columns, q=q, max_rows=most)
        big = rows.index(max(rows))
        assert bool(out[seq[big]].isnan().all())
        verify(c, rows, hq, "bf16", q, out, scale, skip=(big,))
    # a bad page at position 96 of sequence 0 and at 384 of sequence 3 (its last)
    tables = c.dev_tables.clone()
    tables[0, 6] = -1
    tables[3, 24] = c.pages
    _, out, _ = run(luc, c, rows, hq, "bf16", columns=columns, q=q, tables=tables)
    assert bool(out[seq[0]].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(0, 3))
    first = max(0, 384 - (400 - rows[3]))
    assert bool(out[seq[3]][first:].isnan().all())
    assert torch.equal(out[seq[3]][:first], clean[seq[3]][:first])
    # a pool of fewer pages than the tables name
    _, out, _ = run(luc, c, rows, hq, "bf16", columns=columns, q=q, num_blocks=int(c.tables[2, :10].max()))
    assert bool(out[seq[2]].isnan().all())


def test_one_workspace_for_calls_of_other_sizes(luc):
    """Decode, prompt and sparse calls of several sizes in turn on one workspace, and again."""
    calls = [(Cache([3000, 1000], 2, 128, seed=1), [1, 1], 12), (Cache([600], 2, 64, seed=2), [300], 14),
             (Cache([5000], 1, 64, seed=3), [1], 8), (Cache([2000, 30], 2, 128, seed=4), [100, 30], 16)]
    need = max([luc.lib.luc_kv8_workspace_size(len(c.ctx), sum(r), max(r), max(c.ctx), hq, c.hkv, c.d)
                for c, r, hq in calls] + [luc.lib.luc_kv8_sparse_workspace_size(2, 3000, 90, 12, 2, 128)])
    ws = torch.zeros(need // 4, dtype=torch.float32, device="cuda")
    first = [run(luc, c, r, hq, "f16", ws=ws)[1] for c, r, hq in calls]
    chosen = sparse(luc, calls[0][0], 12, "f16", 90, ws=ws)
    for (c, r, hq), was in zip(reversed(calls), reversed(first)):
        q, out, scale = run(luc, c, r, hq, "f16", ws=ws)
        assert torch.equal(out, was)
        verify(c, r, hq, "f16", q, out, scale)
    again = sparse(luc, calls[0][0], 12, "f16", 90, ws=ws)
    assert all(torch.equal(a, b) for a, b in zip(chosen, again))


@pytest.mark.parametrize("rows", [[1, 1, 1], [50, 70, 1], [150, 200, 170]])
def test_another_stream_and_a_captured_call(luc, rows):
    c = Cache([900, 1500, 200], 2, 128, seed=7)
    q, want, scale = run(luc, c, rows, 12, "bf16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert torch.equal(run(luc, c, rows, 12, "bf16", q=q, stream=stream)[1], want)
    total = sum(rows)
    ws = luc.kv8_workspace(3, total, max(rows), 1500, 12, 2, 128)
    out = torch.zeros((total, 12 * 128), dtype=q.dtype, device="cuda")
    q_in = q.clone().contiguous()
    st = torch.tensor([x - r for x, r in zip(c.ctx, rows)], dtype=torch.int32, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        luc.kv8_attention(out, q_in, c.kp, c.vp, c.sp, c.dev_tables, st, 3, total, max(rows), 1500, 1, 2, 12, 2, 128, scale,
                          cu_seqlens=cu, workspace=ws)
    for seed in range(4):
        q_in.copy_(make_q(c, total, 12, "bf16", seed))
        graph.replay()
        eager = run(luc, c, rows, 12, "bf16", q=q_in)[1]
        assert torch.equal(out, eager)


def test_offsets_past_32_bits(luc):
    """A sequence on the last pages of pools of more than 4 GiB."""
    c = Cache([200, 90], 4, 128, seed=6, layers=1, layer=0)
    q, want, scale = run(luc, c, [1, 60], 8, "f16")
    verify(c, [1, 60], 8, "f16", q, want, scale)
    pages, out = sparse(luc, c, 8, "f16", 6)
    more = (1 << 32) // (4 * 2048) + 7
    kp = torch.zeros((more + c.pages, 1, 4, 2048), dtype=torch.uint8, device="cuda")
    vp, sp = torch.zeros_like(kp), torch.zeros((more + c.pages, 1, 4, 2), device="cuda")
    bp = torch.zeros((more + c.pages, 1, 4, 2, 128), dtype=torch.uint8, device="cuda")
    kp[more:], vp[more:], sp[more:], bp[more:] = c.kp, c.vp, c.sp, c.bp
    c.kp, c.vp, c.sp, c.bp, c.pages = kp, vp, sp, bp, more + c.pages
    c.dev_tables = torch.where(c.dev_tables >= 0, c.dev_tables + more, c.dev_tables)
    assert torch.equal(run(luc, c, [1, 60], 8, "f16", q=q)[1], want)
    assert all(torch.equal(a, b) for a, b in zip(sparse(luc, c, 8, "f16", 6), (pages, out)))


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128)])
def test_many_splits(luc, hq, hkv, d):
    """65, 137 and 256 splits of one sequence, under bounds far above it too."""
    c = Cache([16000], hkv, d, seed=2)
    q, out, scale = run(luc, c, [1], hq, "f16")
    verify(c, [1], hq, "f16", q, out, scale)
    for max_ctx in (64 * 1024, 250_000):
        tables = torch.cat([c.dev_tables, torch.full((1, max_ctx // PAGE), -1, dtype=torch.int32, device="cuda")], 1)
        verify(c, [1], hq, "f16", *run(luc, c, [1], hq, "f16", q=q, max_ctx=max_ctx, tables=tables))


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 4), (128, 12, 4)])
def test_longest_first(luc, d, hq, hkv):
    """More workgroups than the chip holds: full splits first, then the rests; sequences without a
    row or a context among them."""
    rng = np.random.default_rng(d)
    ctx = [int(x) for x in rng.integers(1, 2000, 60)] + [6000, 256, 512, 1]
    rows = [1] * 64
    for b in (3, 40):
        rows[b] = 0
    c = Cache(ctx, hkv, d, seed=d, layers=1, layer=0)
    start = [x - r for x, r in zip(c.ctx, rows)]
    start[7] = -5
    q, out, scale = run(luc, c, rows, hq, "bf16", start=start, max_ctx=6000)
    at = sum(rows[:7])
    assert bool(out[at].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(7,))


# ---- chosen pages -----------------------------------------------------------------------------

def sparse(luc, c, hq, dtype, budget, first=1, recent=2, q=None, rows=None, ws=None, stream=None, tables=None, start=None,
           max_ctx=None, scale=None, num_blocks=None, pages=None, seed=1):
    """One row at the end of every context (rows: of those with a 1): (pages, out)."""
    n = len(c.ctx)
    rows = [1] * n if rows is None else rows
    total = sum(rows)
    q = make_q(c, total, hq, dtype, seed) if q is None else q
    cu = None if rows == [1] * n else torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    start = [x - 1 for x in c.ctx] if start is None else start
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    max_ctx = max_ctx or max(c.ctx)
    tables = c.dev_tables if tables is None else tables
    ws = luc.kv8_sparse_workspace(n, max_ctx, budget, hq, c.hkv, c.d) if ws is None else ws
    out = torch.full((total, hq * c.d), 7.0, dtype=DT[dtype], device="cuda")
    scale = c.d ** -0.5 if scale is None else scale
    print(f"  sparse8: ctx {c.ctx[:8]} heads {hq}/{c.hkv}x{c.d} {dtype} budget {budget} ({first}, {recent}) max_ctx {max_ctx}",
          flush=True)
    if pages is None:
        pages = torch.full((n, c.hkv, budget), -9, dtype=torch.int32, device="cuda")
        luc.kv8_select(pages, q, c.bp, c.sp, tables, st, n, max_ctx, first, recent, c.layer, c.layers, hq, c.hkv, c.d,
                       cu_seqlens=cu, workspace=ws, stream=stream, num_blocks=num_blocks)
    luc.kv8_sparse_attention(out, q, c.kp, c.vp, c.sp, tables, st, pages, n, max_ctx, c.layer, c.layers, hq, c.hkv, c.d, scale,
                             cu_seqlens=cu, workspace=ws, stream=stream, num_blocks=num_blocks)
    torch.cuda.synchronize()
    if ws is not None:
        assert not ws[:65536].any(), "arrival counters"
    return pages, out


def want_pages(c, b, h, q, hq, budget, first, recent, bad=()):
    g = hq // c.hkv
    ids = c.tables[b, :-(-c.ctx[b] // PAGE)]
    s = ref.scores(q.double().cpu().numpy().reshape(hq, c.d)[h * g:(h + 1) * g], c.bounds[ids, c.layer, h], c.scales[ids, c.layer, h, 0])
    return ref.choose(s, budget, first, recent, bad)


def verify_sparse(c, hq, dtype, q, pages, out, budget, first=1, recent=2, scale=None, skip=()):
    got = pages.cpu().numpy()
    g = hq // c.hkv
    for b in range(len(c.ctx)):
        if b in skip:
            continue
        for h in range(c.hkv):
            assert got[b, h].tolist() == want_pages(c, b, h, q[b], hq, budget, first, recent), (b, h)
            at = torch.tensor([p for p in got[b, h] if p >= 0], device="cuda")
            pos = (at[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(-1)
            pos = pos[pos < c.ctx[b]]
            heads = slice(h * g, (h + 1) * g)
            want, tol = ref.attention(q[b].double().view(1, hq, c.d)[:, heads], c.k[b][pos, h:h + 1], c.v[b][pos, h:h + 1],
                                      torch.ones(1, len(pos), dtype=torch.bool, device="cuda"),
                                      c.d ** -0.5 if scale is None else scale, DT[dtype])
            serving_ref.check(out[b].view(1, hq, c.d)[:, heads], want, tol, DT[dtype], f"sequence {b} head {h} of {c.ctx[b]}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS[:7])
def test_choices_and_attention_over_them(luc, hq, hkv, d, dtype):
    """Budgets below, at and above a context's pages; contexts that end inside a page."""
    c = Cache([1, 16, 17, 129, 700, 2500], hkv, d, seed=hq, spread=2)
    q = make_q(c, 6, hq, dtype)
    for budget, first, recent in ((8, 1, 2), (3, 1, 2), (9, 0, 1), (44, 3, 5), (200, 1, 2), (1, 0, 1)):
        pages, out = sparse(luc, c, hq, dtype, budget, first, recent, q=q)
        verify_sparse(c, hq, dtype, q, pages, out, budget, first, recent)
        if budget == 200:  # everything
            dense = run(luc, c, [1] * 6, hq, dtype, q=q)[1]
            err = (dense.double() - out.double()).abs().max() / out.double().abs().max()
            assert float(err) <= 2 * torch.finfo(DT[dtype]).eps


@pytest.mark.parametrize("d", [64, 128])
def test_equal_scores(luc, d):
    """Pages that share their bounds, queries of zeros, of NaN and of infinities: the lower page."""
    c = Cache([1600, 1000], 2, d, seed=1)
    for b in range(2):
        ids = c.tables[b, :-(-c.ctx[b] // PAGE)]
        c.bounds[ids, 1] = c.bounds[ids[0], 1]
        c.scales[ids, 1, :, 0] = 2.0 ** (np.arange(len(ids)) // 7 % 3)[:, None]
    c.bp, c.sp = torch.from_numpy(c.bounds).cuda(), torch.from_numpy(c.scales).cuda()
    q = make_q(c, 2, 8, "f16")
    for i, x in enumerate((None, 0.0, float("nan"), float("inf"), -float("inf"))):
        if x is not None:
            q[0], q[1, ::3] = x, x
        pages, _ = sparse(luc, c, 8, "f16", 20, q=q)
        got = pages.cpu().numpy()
        for b in range(2):
            for h in range(2):
                assert got[b, h].tolist() == want_pages(c, b, h, q[b], 8, 20, 1, 2), (i, b, h)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_codes_are_rounded_to_units(luc, d, dtype):
    """A query of one dimension: pages whose bounds there are every code, in any order; what decides is the code's
    nearest whole number, halves to the even one, and of equal ones the lower page."""
    codes = np.random.default_rng(d).permutation(np.delete(np.arange(256), [127, 255]))
    c = Cache([254 * PAGE], 2, d, seed=1)
    ids = c.tables[0]
    c.scales[ids, 1, :, 0] = 0.25
    c.sp = torch.from_numpy(c.scales).cuda()
    for dim, value in ((5, 1.0), (37, -3.0), (d - 1, 0.5), (16, -1e-3)):
        c.bounds[:] = 0
        c.bounds[ids, 1, :, 0 if value > 0 else 1, dim] = codes[:, None]
        c.bp = torch.from_numpy(c.bounds).cuda()
        q = torch.zeros(1, 6 * d, dtype=DT[dtype], device="cuda")
        q.view(6, d)[[0, 1, 2, 4], dim] = value
        for budget in (3, 20, 60, 100, 128, 150, 180, 220, 253):
            pages, _ = sparse(luc, c, 6, dtype, budget, 0, 1, q=q)
            for h in range(2):
                assert pages[0, h].tolist() == want_pages(c, 0, h, q[0], 6, budget, 0, 1), (dim, budget, h)


def test_many_pages(luc):
    """More pages than a workgroup keeps keys of, and scores of both signs over many powers of two."""
    hkv, d, n = 1, 64, 8300
    rng = np.random.default_rng(0)
    c = Cache([n * PAGE - 5], hkv, d, seed=8, layers=1, layer=0)
    x = rng.standard_normal((n, 2, d)) * 2.0 ** rng.integers(-3, 9, (n, 1, 1))
    ids = c.tables[0]
    c.bounds[ids, 0, 0] = ref.encode(np.clip(x, -448, 448))
    c.bp = torch.from_numpy(c.bounds).cuda()
    q = make_q(c, 1, 4, "bf16")
    for budget in (3, 64, 1000, 8299):
        pages, out = sparse(luc, c, 4, "bf16", budget, q=q)
        assert pages[0, 0].tolist() == want_pages(c, 0, 0, q[0], 4, budget, 1, 2), budget
        assert bool(out.isfinite().all())


@pytest.mark.parametrize("d", [64, 128])
def test_batches_with_rows_left_out(luc, d):
    """Sequences without a row, beyond max_ctx, at no position; pages outside the pool come last, and a row
    that reads one is NaN; rows of nobody stay."""
    c = Cache([900, 400, 700, 1300, 60], 2, d, seed=2)
    hq, budget = 6, 12
    q = make_q(c, 5, hq, "bf16")
    pages, clean = sparse(luc, c, hq, "bf16", budget, q=q)
    verify_sparse(c, hq, "bf16", q, pages, clean, budget)
    some = [1, 0, 1, 1, 0]
    got, out = sparse(luc, c, hq, "bf16", budget, q=q[[0, 2, 3]], rows=some)
    assert bool((got[[1, 4]] == -1).all()) and torch.equal(got[[0, 2, 3]], pages[[0, 2, 3]])
    assert torch.equal(out, clean[[0, 2, 3]])
    # two rows of a sequence are more than the calls have
    got, out = sparse(luc, c, hq, "bf16", budget, q=q, rows=[1, 2, 0, 1, 1], start=[899, 398, 699, 1299, 59])
    assert bool((got[1] == -1).all()) and bool(out[1:3].isnan().all())
    assert torch.equal(out[[0, 3, 4]], clean[[0, 3, 4]]) and torch.equal(got[[0, 3, 4]], pages[[0, 3, 4]])
    got, out = sparse(luc, c, hq, "bf16", budget, q=q, max_ctx=1000)
    assert bool((got[3] == -1).all()) and bool(out[3].isnan().all()) and torch.equal(out[:3], clean[:3])
    got, out = sparse(luc, c, hq, "bf16", budget, q=q, start=[899, -1, 699, -(1 << 31), 59])
    assert bool((got[[1, 3]] == -1).all()) and bool(out[[1, 3]].isnan().all()) and torch.equal(out[[0, 2, 4]], clean[[0, 2, 4]])
    tables = c.dev_tables.clone()
    bad = [p for p in pages[0, 0].tolist() if 2 <= p < 54][:1]
    tables[0, bad[0]] = c.pages
    tables[2, 0] = -3  # the first page: always chosen
    got, out = sparse(luc, c, hq, "bf16", budget, q=q, tables=tables)
    for h in range(2):
        assert got[0, h].tolist() == want_pages(c, 0, h, q[0], hq, budget, 1, 2, bad)
    assert bool(out[0].isfinite().all()) and bool(out[2].isnan().all()) and torch.equal(out[[1, 3, 4]], clean[[1, 3, 4]])


@pytest.mark.parametrize("d", [64, 128])
def test_lists_that_are_no_choice(luc, d):
    """Attention over given lists: any ascending one is right, and what is outside the context is NaN."""
    c = Cache([900, 300], 2, d, seed=3)
    hq, budget = 8, 6
    q = make_q(c, 2, hq, "f16")
    good = torch.tensor([[[0, 3, 9, 20, 40, 56]] * 2, [[1, 2, 4, 6, 8, 18]] * 2], dtype=torch.int32, device="cuda")
    _, clean = sparse(luc, c, hq, "f16", budget, q=q, pages=good)
    for b in range(2):
        pos = (good[b, 0].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(-1)
        pos = pos[pos < c.ctx[b]]
        want, tol = ref.attention(q[b].double().view(1, hq, d), c.k[b][pos], c.v[b][pos],
                                  torch.ones(1, len(pos), dtype=torch.bool, device="cuda"), d ** -0.5, torch.float16)
        serving_ref.check(clean[b].view(1, hq, d), want, tol, torch.float16, f"sequence {b}")
    for at, value in ((5, 55), (5, 57), (2, -1), (2, 56), (0, 1 << 30), (3, -(1 << 31))):
        lists = good.clone()
        lists[0, 1, at] = value
        _, out = sparse(luc, c, hq, "f16", budget, q=q, pages=lists)
        o, w = out.view(2, hq, d), clean.view(2, hq, d)
        assert bool(o[0, 4:].isnan().all()), (at, value)
        assert torch.equal(o[0, :4], w[0, :4]) and torch.equal(o[1], w[1])


def test_sparse_on_another_stream_and_captured(luc):
    c = Cache([2000, 5000, 333], 2, 128, seed=7)
    hq, budget = 12, 40
    q = make_q(c, 3, hq, "bf16")
    want = sparse(luc, c, hq, "bf16", budget, q=q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = sparse(luc, c, hq, "bf16", budget, q=q, stream=stream)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    ws = luc.kv8_sparse_workspace(3, 5000, budget, hq, 2, 128)
    out = torch.zeros(3, hq * 128, dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(3, 2, budget, dtype=torch.int32, device="cuda")
    st = torch.tensor([x - 1 for x in c.ctx], dtype=torch.int32, device="cuda")
    q_in = q.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        luc.kv8_select(pages, q_in, c.bp, c.sp, c.dev_tables, st, 3, 5000, 1, 2, 1, 2, hq, 2, 128, workspace=ws)
        luc.kv8_sparse_attention(out, q_in, c.kp, c.vp, c.sp, c.dev_tables, st, pages, 3, 5000, 1, 2, hq, 2, 128, 128 ** -0.5,
                                 workspace=ws)
    for seed in range(5):
        q_in.copy_(make_q(c, 3, hq, "bf16", seed))
        graph.replay()
        p, o = sparse(luc, c, hq, "bf16", budget, q=q_in)
        assert torch.equal(p, pages) and torch.equal(o, out)
