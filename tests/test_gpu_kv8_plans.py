"""The 8-bit cache's attention and page selection at sizes that reach every plan of their launches: many splits and their
merge, splits longer than a batch of page numbers, reversed orders of chunks, several tiles of pages a wave."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
import serving_ref
from test_gpu_kv8_attention import DT, PAGE, Cache, make_q, run, verify

pytestmark = pytest.mark.gpu


class LongContext:
    """One sequence of one kv head (a Cache, made on the GPU), every byte behind its end NaN.  V has a mean, of either sign for
    every 2048 tokens: a part of a context that is left out, or counted twice, shows."""

    def __init__(self, n, d, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.hkv, self.d, self.layers, self.layer = [n], 1, d, 1, 0
        count = -(-n // PAGE)
        self.pages = count + 1
        ids = torch.randperm(self.pages, generator=gen, device="cuda")[:count]
        self.dev_tables = ids.to(torch.int32)[None]
        self.tables = self.dev_tables.cpu().numpy()
        self.sp = torch.full((self.pages, 1, 1, 2), float("nan"), device="cuda")
        self.k, self.v = [], []
        pools = []
        for is_v, keep in enumerate((self.k, self.v)):
            x = torch.randn(count, PAGE, d, generator=gen, device="cuda") * 80
            if is_v:
                sign = torch.randint(0, 2, (count // 128 + 1,), generator=gen, device="cuda") * 2.0 - 1
                x += 100 * sign.repeat_interleave(128)[:count, None, None]
            codes = x.clamp(-448, 448).to(torch.float8_e4m3fn)
            e = torch.randint(-8, -6 if is_v else -5, (count,), generator=gen, device="cuda").float()
            self.sp[ids, 0, 0, is_v] = 2.0 ** e
            keep.append((codes.double() * (2.0 ** e.double())[:, None, None]).view(-1, 1, d)[:n])
            raw = codes.view(torch.uint8).clone()
            raw.view(-1, d)[n:] = 0x7F
            pool = torch.full((self.pages, 1, 1, 16 * d), 0xFF, dtype=torch.uint8, device="cuda")
            pool[ids, 0, 0] = (raw.view(count, 4, 4, d).transpose(2, 3) if is_v else raw).reshape(count, 16 * d)
            pools.append(pool)
        self.kp, self.vp = pools


def splits_of(luc, batch, rows, max_ctx, hq, hkv, d, tiles=1):
    """Splits of a decode step, from its workspace: counters, then (m, l) and o of 8 columns a split."""
    size = luc.lib.luc_kv8_workspace_size(batch, rows, 1, max_ctx, hq, hkv, d)
    for splits in range(1, 257):
        n = batch * hkv * tiles * splits * 8
        if size == (1 << 18) + -(-n * 8 // 256) * 256 + n * d * 4:
            return splits
    return 1 if size == 0 else None


def verify_long(c, hq, dtype, q, out, scale, split_tokens):
    """verify() of one row, with the f32 sums as they are made: over a split's tokens, then its waves' halves and up to 256
    splits, not over the whole context."""
    args = [x.view(1, hq, c.d) for x in (q[0].double(), out[0])]
    seen = torch.ones(1, c.ctx[0], dtype=torch.bool, device="cuda")
    want, tol = ref.attention(args[0], c.k[0], c.v[0], seen, scale, DT[dtype])
    size, _ = ref.attention(args[0], c.k[0], c.v[0].abs(), seen, scale, DT[dtype])
    terms = split_tokens + 8 + 256
    assert terms < c.ctx[0]
    tol = tol - (c.ctx[0] - terms) * 2.0 ** -24 * size
    one_split = 2048 / c.ctx[0] * size.median()  # (what a split more or less is worth, about)
    assert float(tol.max()) < float(one_split) / 4
    serving_ref.check(args[1], want, tol, DT[dtype], f"{c.ctx[0]} tokens")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,n,splits", [(64, 131_073, 65), (64, 262_200, 129), (64, 393_300, 193), (64, 524_288, 256),
                                        (128, 140_001, 73), (128, 524_289, 241)])
def test_splits_beyond_a_wave(luc, d, n, splits, dtype):
    """Contexts of more splits than a wave has lanes, and of every place among four times as many."""
    assert splits_of(luc, 1, 1, n, 5, 1, d) == splits
    c = LongContext(n, d, seed=splits)
    tokens = -(-n // (splits - 1))  # of a split, at most
    q, out, scale = run(luc, c, [1], 5, dtype, q_std=0.5)
    verify_long(c, 5, dtype, q, out, scale, tokens)
    # a shorter context of the same plan
    short = LongContext(n // 3, d, seed=splits + 1)
    tables = torch.cat([short.dev_tables, torch.full((1, n // PAGE + 1), -1, dtype=torch.int32, device="cuda")], 1)
    q, out, scale = run(luc, short, [1], 5, dtype, max_ctx=n, tables=tables, q_std=0.5)
    verify_long(short, 5, dtype, q, out, scale, tokens)


def verify_rows(c, b, first, rows, hq, dtype, q, out, scale, r0):
    """Of sequence b, whose rows begin at row r0 and position `first`, the rows `rows`."""
    at = torch.tensor(rows, device="cuda")
    seen = torch.arange(c.ctx[b], device="cuda")[None] <= (first + at)[:, None]
    want, tol = ref.attention(q[r0 + at].double().view(len(rows), hq, c.d), c.k[b], c.v[b], seen, scale, DT[dtype])
    serving_ref.check(out[r0 + at].view(len(rows), hq, c.d), want, tol, DT[dtype], f"sequence {b}, rows {rows[:4]}..")


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, "bf16"), (12, 2, 128, "f16")])
def test_one_split_of_many_pages(luc, hq, hkv, d, dtype):
    """A prompt of more than 4096 rows from an empty cache, in one split, whose waves look up page numbers more than once; and
    pages outside the pool among the first of them and behind."""
    n = 4803
    assert luc.lib.luc_kv8_workspace_size(1, n, n, n, hq, hkv, d) == 0
    c = Cache([n], hkv, d, seed=d, layers=1, layer=0)
    q, clean, scale = run(luc, c, [n], hq, dtype)
    rows = list(range(0, 40)) + list(range(4050, 4180)) + list(range(n - 150, n)) + list(range(40, 4050, 97))
    verify_rows(c, 0, 0, rows, hq, dtype, q, clean, scale, 0)
    for bad in ((270, 285), (259,), (299,), (31, 290)):  # pages
        tables = c.dev_tables.clone()
        for i, p in enumerate(bad):
            tables[0, p] = (-1, c.pages)[i % 2]
        _, out, _ = run(luc, c, [n], hq, dtype, q=q, tables=tables)
        first = min(bad) * PAGE
        assert torch.equal(out[:first], clean[:first]) and bool(out[first:].isnan().all()), bad


@pytest.mark.parametrize("hq,hkv,d,dtype,rows,held", [
    (14, 2, 64, "bf16", [2048, 1531, 1702, 1999], [0, 0, 0, 0]), (28, 4, 128, "f16", [1900, 701, 1402], [0, 100, 33]),
    (8, 8, 64, "f16", [900, 1700, 1111, 40, 1], [3, 0, 17, 0, 5])])
def test_chunks_in_reversed_order(luc, hq, hkv, d, dtype, rows, held):
    """Two rounds of workgroups and more, the last of them not full: every other round has its chunks in reverse."""
    group, cols = hq // hkv, 128 if d == 64 else 256
    n = len(rows) * hkv * -(-max(rows) * group // cols)
    assert n >= 512 and n % 256
    c = Cache([r + h for r, h in zip(rows, held)], hkv, d, seed=d, layers=1, layer=0)
    q, out, scale = run(luc, c, rows, hq, dtype, tail=2)
    at = 0
    for b, (r, h) in enumerate(zip(rows, held)):
        some = sorted({x for i in range(0, r, 50) for x in (i, min(i + 17, r - 1))} | {r - 1})
        verify_rows(c, b, h, some, hq, dtype, q, out, scale, at)
        assert bool(out[at:at + r].isfinite().all())
        at += r


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 4), (128, 12, 4)])
def test_longest_first_of_whole_splits(luc, d, hq, hkv):
    """Contexts that end with a split, just before and just behind, some of several splits; sequences without a row or a
    context among them."""
    rng = np.random.default_rng(d)
    ctx = [2048, 4096, 6144, 2047, 2049, 4095, 4097, 6100, 1, 4096, 2048, 6143] + [int(x) for x in rng.integers(1, 6144, 52)]
    rows = [1] * 64
    for b in (1, 30):
        rows[b] = 0
    assert splits_of(luc, 64, 62, 6144, hq, hkv, d) == 3   # of 2048 tokens, more than two workgroups a CU
    c = Cache(ctx, hkv, d, seed=d, layers=1, layer=0)
    start = [x - r for x, r in zip(c.ctx, rows)]
    start[5], start[9] = -5, 9000
    q, out, scale = run(luc, c, rows, hq, "bf16", start=start, max_ctx=6144)
    for b in (5, 9):
        assert bool(out[sum(rows[:b])].isnan().all())
    verify(c, rows, hq, "bf16", q, out, scale, skip=(5, 9))


def test_prompts_past_32_bits(luc):
    """Prompts on the last pages of pools of more than 4 GiB, by the kernel for many columns."""
    rows, ctx = [300, 160], [500, 160]
    c = Cache(ctx, 4, 128, seed=6, layers=1, layer=0)
    q, want, scale = run(luc, c, rows, 8, "f16", columns=True)
    verify(c, rows, 8, "f16", q, want, scale)
    more = (1 << 32) // (4 * 2048) + 7
    kp = torch.zeros((more + c.pages, 1, 4, 2048), dtype=torch.uint8, device="cuda")
    vp, sp = torch.zeros_like(kp), torch.zeros((more + c.pages, 1, 4, 2), device="cuda")
    kp[more:], vp[more:], sp[more:] = c.kp, c.vp, c.sp
    c.kp, c.vp, c.sp, c.pages = kp, vp, sp, more + c.pages
    c.dev_tables = torch.where(c.dev_tables >= 0, c.dev_tables + more, c.dev_tables)
    assert torch.equal(run(luc, c, rows, 8, "f16", q=q, columns=True)[1][:sum(rows)], want[:sum(rows)])


# ---- the choice of pages ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("batch,hq,hkv,d,most,tiles", [(32, 8, 4, 64, 500, 2), (32, 16, 4, 128, 801, 4), (64, 28, 4, 128, 1024, 8),
                                                       (64, 16, 8, 64, 1023, 16), (64, 8, 8, 128, 2100, 16)])
def test_choices_of_full_batches(luc, batch, hq, hkv, d, most, tiles, dtype):
    """Waves that score several tiles of 16 pages: contexts of a page more than the budget up to `most` pages, that end inside a
    tile, with one, and a page behind those of a wave or of a workgroup."""
    t = 1  # the launch's rule: no more than 512 workgroups of 64 pages each, or more pages up to 16 times as many
    while t < 16 and batch * hkv * -(-(-(-most // 4) * 4) // (64 * t)) > 512:
        t *= 2
    assert t == tiles
    budget, first, recent = 24, 1, 2
    rng = np.random.default_rng(most)
    edges = [x for k in (1, 2, 3, 4, 5, 7, 8, 16) for x in (16 * k * tiles - 1, 16 * k * tiles, 16 * k * tiles + 1)] + [25, 24, 26, 63, 64, 65]
    pages = [most] + [x for x in edges if 0 < x <= most][:batch - 8]
    pages += [int(x) for x in rng.integers(1, most + 1, batch - len(pages))]
    ctx = [16 * p - int(rng.integers(0, 16)) for p in pages]
    total = sum(pages)
    perm = rng.permutation(total + 2).astype(np.int32)
    tables = np.full((batch, most), -7, np.int32)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = perm[at:at + n]
        at += n
    hi = rng.standard_normal((total + 2, 1, hkv, d), dtype=np.float32) * 60
    codes = torch.from_numpy(np.stack([hi, hi - np.abs(rng.standard_normal(hi.shape, dtype=np.float32)) * 90], 3).clip(-448, 448))
    bounds = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.from_numpy(2.0 ** rng.integers(-9, -6, (total + 2, 1, hkv, 2)).astype(np.float32))
    q = (torch.randn(batch, hq * d, generator=torch.Generator().manual_seed(most)) * 1.4).to(DT[dtype])
    got = torch.full((batch, hkv, budget), -9, dtype=torch.int32, device="cuda")
    ws = luc.kv8_sparse_workspace(batch, 16 * most, budget, hq, hkv, d)
    start = torch.tensor([x - 1 for x in ctx], dtype=torch.int32, device="cuda")
    print(f"  select8: batch {batch} heads {hq}/{hkv}x{d} {dtype} up to {most} pages", flush=True)
    for _ in range(2):
        luc.kv8_select(got, q.cuda(), bounds.cuda(), scales.cuda(), torch.from_numpy(tables).cuda(), start, batch, 16 * most, first,
                       recent, 0, 1, hq, hkv, d, workspace=ws)
        torch.cuda.synchronize()
    assert not ws[:65536].any(), "arrival counters"
    got, group = got.cpu().numpy(), hq // hkv
    x, bounds, scales = q.double().numpy().reshape(batch, hq, d), bounds.numpy(), scales.numpy()
    for b in range(batch):
        ids = tables[b, :pages[b]]
        for h in range(hkv):
            s = ref.scores(x[b, h * group:(h + 1) * group], bounds[ids, 0, h], scales[ids, 0, h, 0])
            assert got[b, h].tolist() == ref.choose(s, budget, first, recent), (b, h, pages[b])
