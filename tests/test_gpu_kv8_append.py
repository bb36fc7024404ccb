"""luc_kv8_append and luc_kv8_read: q has the bits of luc_qk_norm_rope_append, pools, scales and key bounds those of the
format written page by page from the k and v that the 16-bit append stores."""
import numpy as np
import pytest
import torch

import kv8_ref as ref

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
HEADS = [(14, 2, 64), (28, 4, 128), (5, 1, 128), (8, 8, 64)]


def rope(max_pos, d):
    i = np.arange(d // 2) * 2.0 / d
    th = np.arange(max_pos)[:, None] / 1e6 ** i[None]
    return (torch.from_numpy(np.cos(th).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(th).astype(np.float32)).cuda())


class Book:
    """8-bit pools on the device, the same on the host, and 16-bit pools beside them.  lead: every call is one of many
    rows, of which so many without a slot come before, and more behind."""

    def __init__(self, luc, hq, hkv, d, dtype, pages=12, layers=2, layer=1, bias=True, norm=True, seed=0, bounds=True,
                 fill=0xFF, lead=None):
        self.lead = lead
        self.luc, self.hq, self.hkv, self.d, self.dt, self.layers, self.layer = luc, hq, hkv, d, DT[dtype], layers, layer
        self.gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=self.gen)  # noqa: E731
        self.host = ref.Pools(pages, layers, hkv, d, fill, scale=2.0 ** 7)  # (of earlier sequences)
        self.k, self.v, self.scales, self.bounds = self.host.device()
        self.with_bounds = bounds
        self.pages = pages
        self.cos, self.sin = rope(400, d)
        a, b = hq * d, (hq + hkv) * d
        self.kw = {}
        if bias:
            x = (rnd((hq + 2 * hkv) * d) * 0.3).to(self.dt).cuda()
            self.kw.update(q_bias=x[:a], k_bias=x[a:b], v_bias=x[b:])
        if norm:
            self.kw.update(q_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda(), k_norm=(1 + 0.2 * rnd(d)).to(self.dt).cuda())

    def rows(self, n, k_scale=1.4, v_scale=1.0, extra=0):
        a, b = self.hq * self.d, (self.hq + self.hkv) * self.d
        x = torch.randn(n, b + self.hkv * self.d + extra, generator=self.gen)
        x[:, a:b] *= k_scale
        x[:, b:] *= v_scale
        return x.to(self.dt).cuda()

    def append(self, slots, pos, qkv, in_place=False, num_blocks=None):
        """One call, checked against the host."""
        if self.lead is not None:
            pad = self.rows(self.lead + 600, extra=qkv.shape[1] - (self.hq + 2 * self.hkv) * self.d)
            qkv = torch.cat([pad[:self.lead], qkv, pad[self.lead:]])
            slots = [-1] * self.lead + [int(x) for x in slots] + [-1] * 600
            pos = [3] * self.lead + list(pos) + [-1] * 50 + [9] * 550
        n, a, b, c = len(slots), self.hq * self.d, (self.hq + self.hkv) * self.d, (self.hq + 2 * self.hkv) * self.d
        q, k, v = qkv[:, :a], qkv[:, a:b], qkv[:, b:c]
        sl = torch.tensor(slots, dtype=torch.int64, device="cuda")
        ps = torch.tensor(pos, dtype=torch.int32, device="cuda")
        shape = (self.pages, self.layers, self.hkv, PAGE, self.d)
        kp, vp = (torch.zeros(shape, dtype=self.dt, device="cuda") for _ in range(2))
        want_q, got_q = (torch.full((n, a + 8), 7.0, dtype=self.dt, device="cuda") for _ in range(2))
        args = (self.layer, self.layers, self.hq, self.hkv, self.d)
        self.luc.qk_norm_rope_append(q, k, v, self.cos, self.sin, ps, sl, kp, vp, *args, q_out=want_q[:, :a],
                                     num_blocks=num_blocks, **self.kw)
        print(f"  append8: rows {n} heads {self.hq}/{self.hkv}x{self.d} {self.dt} slots {slots[:6]}", flush=True)
        if in_place:
            want_q[:, :a] = torch.where(((ps >= 0) & (ps < 400))[:, None], want_q[:, :a], q)  # (the others' q stays)
            qkv = qkv.clone()
            q, k, v = qkv[:, :a], qkv[:, a:b], qkv[:, b:c]
        self.luc.kv8_append(q, k, v, self.cos, self.sin, ps, sl, self.k, self.v, self.scales, *args,
                            bounds=self.bounds if self.with_bounds else None, q_out=None if in_place else got_q[:, :a],
                            num_blocks=num_blocks, **self.kw)
        torch.cuda.synchronize()
        assert torch.equal((q if in_place else got_q[:, :a]).view(torch.int16), want_q[:, :a].view(torch.int16)) or \
            not in_place and torch.equal(got_q, want_q)
        assert bool((got_q[:, a:] == 7).all())
        usable = (num_blocks or self.pages) * PAGE
        live = [i for i in range(n) if 0 <= slots[i] < usable and 0 <= pos[i] < 400]
        page, off = np.array(slots)[live] // PAGE, np.array(slots)[live] % PAGE
        kx, vx = (p[torch.from_numpy(page).cuda(), self.layer, :, torch.from_numpy(off).cuda()].double().cpu().numpy()
                  for p in (kp, vp))
        self.host.append(self.layer, [slots[i] for i in live], kx, vx)
        self.check()

    def check(self):
        assert np.array_equal(self.scales.cpu().numpy(), self.host.scales)
        for name, got, want in (("k", self.k, self.host.k), ("v", self.v, self.host.v), ("bounds", self.bounds, self.host.bounds)):
            if name != "bounds" or self.with_bounds:
                assert ref.equal_codes(got.cpu().numpy(), want), name


def seq(table, start, n):
    pos = list(range(start, start + n))
    return [table[p // PAGE] * PAGE + p % PAGE for p in pos], pos


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lead", [None, 0, 13])
def test_prompts_and_steps(luc, hq, hkv, d, dtype, lead):
    """Prompts of odd lengths, then rows one by one, several, and up to a page's end, louder and quieter than what
    the pages hold; a page that is taken by another sequence."""
    book = Book(luc, hq, hkv, d, dtype, seed=d + hq, lead=lead)
    a, b = [7, 2, 9, 0, 4], [11, 1, 5]
    for n_a, start_a, n_b, start_b, k_scale, v_scale in (
            (33, 0, 17, 0, 1.4, 1.0), (1, 33, 1, 17, 1.4, 1.0), (1, 34, 1, 18, 9.0, 40.0), (3, 35, 13, 19, 100.0, 0.01),
            (10, 38, 1, 32, 0.001, 2.0), (17, 48, 2, 33, 3.0, 3000.0)):
        (sa, pa), (sb, pb) = seq(a, start_a, n_a), seq(b, start_b, n_b)
        book.append(sa + sb, pa + pb, book.rows(n_a + n_b, k_scale, v_scale, extra=8))
    s, p = seq([9, 1], 0, 20)  # pages of others, anew
    book.append(s, p, book.rows(20, 0.05, 0.05), in_place=True)


@pytest.mark.parametrize("hq,hkv,d", HEADS[:2])
@pytest.mark.parametrize("norm,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("lead", [None, 7])
def test_norms_and_biases(luc, hq, hkv, d, norm, bias, lead):
    book = Book(luc, hq, hkv, d, "bf16", norm=norm, bias=bias, bounds=norm, lead=lead)
    s, p = seq([3, 8, 1, 5], 5, 50)
    book.append(s, p, book.rows(50))
    for i in range(55, 60):
        s, p = seq([3, 8, 1, 5], i, 1)
        book.append(s, p, book.rows(1, 2.0 ** (i - 55)))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_values_at_the_edges(luc, dtype):
    """Infinities and NaN, zeros, values beyond the limit, subnormals of the type, and largest values at and next to
    448 times a power of two."""
    book = Book(luc, 4, 2, 64, dtype, norm=False, bias=False)
    qkv = book.rows(16)
    k, v = qkv[:, 256:384], qkv[:, 384:]
    tiny = torch.finfo(book.dt).smallest_normal
    v[0, 3], v[0, 70], v[1, 5], v[2, 80] = float("nan"), float("inf"), -float("inf"), float("nan")
    k[3, 4] = float("nan")  # (its partner too, rotated)
    k[4], v[4] = 0, 0
    v[5, :64], v[6, 64:] = 65504.0, -61000.0
    book.append(*seq([2], 0, 7), qkv[:7])
    v[7:] = v[7:] * 0
    for i, x in enumerate((448.0, 449.0, 3.5, 3.515625, 1.75, tiny, tiny / 8, 57344.0, 57376.0)):
        v[7 + i, i], v[7 + i, 64 + i] = x, -x
        book.append(*seq([4 + i // 4], i % 4, 1), qkv[7 + i:8 + i])


@pytest.mark.parametrize("lead", [None, 15])
def test_rows_that_have_no_place(luc, lead):
    """Slots and positions of no page and no table: the rows' q, or nothing, and no cache."""
    book = Book(luc, 14, 2, 64, "f16", lead=lead)
    slots = [-1, 37, 38, 12 * PAGE, 39, -(1 << 40), 1 << 40, 96, 97, 98]
    pos = [5, 6, 7, 8, 9, 10, 11, 399, 400, -1]
    book.append(slots, pos, book.rows(10))
    # a page whose first row, or one in between, has no position
    book.append([7 * PAGE, 7 * PAGE + 1, 7 * PAGE + 2, 8 * PAGE, 7 * PAGE + 3, 8 * PAGE + 1], [400, 1, -1, -7, 2, 3], book.rows(6))
    # a pool of fewer pages than the tensors hold
    s, p = seq([5, 6], 12, 9)
    book.append(s, p, book.rows(9), num_blocks=6)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("lead", [None, 0, 1, 11, 16, 31])
def test_rows_in_any_order(luc, hq, hkv, d, lead):
    """Rows of a page in descending order, with others and padding between them, as far apart as they may be."""
    book = Book(luc, hq, hkv, d, "bf16", lead=lead)
    s, p = seq([2, 7], 0, 32)
    book.append(s[::-1], p[::-1], book.rows(32))
    # two pages row by row, and one of them again at other offsets, 31 rows behind the first
    s = [x for i in range(15) for x in (5 * PAGE + i, 6 * PAGE + 15 - i)] + [-1, 5 * PAGE + 15]
    book.append(s, [x % PAGE + 3 for x in s[:-2]] + [1, 7], book.rows(32))
    # joined at offsets with gaps
    book.append([5 * PAGE + 9, 2 * PAGE + 3, -1, 5 * PAGE + 4, 2 * PAGE + 1, 5 * PAGE + 14], [1, 2, 3, 4, 5, 6], book.rows(6, 30.0, 9.0))
    s = np.random.default_rng(0).permutation(16) + 9 * PAGE
    book.append(s.tolist() + [8 * PAGE], [30] * 17, book.rows(17))


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("lead", [None, 5])
def test_many_rows(luc, hq, hkv, d, lead):
    """A batch of single rows and ragged prompts beyond what one workgroup has."""
    book = Book(luc, hq, hkv, d, "bf16", pages=90, layers=1, layer=0, lead=lead)
    perm = np.random.default_rng(1).permutation(90).tolist()
    s, p = [], []
    for i, n in enumerate((100, 1, 16, 31, 64)):
        x = seq(perm[10 * i:], 0, n)
        s, p = s + x[0], p + x[1]
    book.append(s, p, book.rows(len(s)))
    single = [seq([perm[50 + i]], i % 16, 1) for i in range(40)]
    book.append([x[0][0] for x in single], [x[1][0] for x in single], book.rows(40))


def test_offsets_past_32_bits(luc):
    """The last pages of pools of more than 4 GiB: appended and read."""
    d, hkv = 128, 4
    pages = (1 << 32) // (hkv * 16 * d) + 3
    kp = torch.zeros((pages, 1, hkv, 16 * d), dtype=torch.uint8, device="cuda")
    vp, scales = torch.zeros_like(kp), torch.zeros((pages, 1, hkv, 2), device="cuda")
    book = Book(luc, 4, 4, d, "bf16", pages=3, layers=1, layer=0, norm=False)
    s, p = seq([2, 0, 1], 0, 40)
    qkv = book.rows(40)
    book.append(s, p, qkv)
    a, b = 4 * d, 8 * d
    slots = torch.tensor(s, device="cuda") + (pages - 3) * PAGE
    luc.kv8_append(qkv[:, :a].contiguous().expand(40, a), qkv[:, a:b].contiguous(), qkv[:, b:].contiguous(), book.cos, book.sin,
                   torch.tensor(p, dtype=torch.int32, device="cuda"), slots, kp, vp, scales, 0, 1, 4, 4, d, **book.kw)
    k_out, v_out = (torch.zeros(40, hkv * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    luc.kv8_read(k_out, v_out, slots, kp, vp, scales, 0, 1, hkv, d)
    want = [torch.from_numpy(book.host.values([2, 0, 1], 0, is_v)[:40]).view(40, -1).bfloat16() for is_v in (False, True)]
    assert torch.equal(k_out.cpu(), want[0]) and torch.equal(v_out.cpu(), want[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hkv,d", [(2, 64), (4, 128), (1, 128), (8, 64)])
def test_read(luc, hkv, d, dtype):
    """Every code under scales of all sizes, in any order, to padded rows; rows without a slot stay."""
    rng = np.random.default_rng(d + hkv)
    host = ref.Pools(9, 2, hkv, d)
    host.k[:], host.v[:] = rng.integers(0, 256, host.k.shape), rng.integers(0, 256, host.v.shape)
    host.scales[:] = 2.0 ** rng.integers(-30, 8, host.scales.shape)
    k, v, scales, _ = host.device()
    n = 300
    slots = rng.integers(0, 9 * PAGE, n)
    slots[[3, 77, 299]] = -1, 9 * PAGE, -(1 << 50)
    dt = DT[dtype]
    outs = [torch.full((n, hkv * d + 8), 7.0, dtype=dt, device="cuda") for _ in range(2)]
    dev = torch.from_numpy(slots).cuda()
    luc.kv8_read(outs[0][:, :hkv * d], outs[1][:, :hkv * d], dev, k, v, scales, 1, 2, hkv, d)
    torch.cuda.synchronize()
    ok = (slots >= 0) & (slots < 9 * PAGE)
    for out, is_v in zip(outs, (False, True)):
        want = torch.from_numpy(host.values(range(9), 1, is_v)[np.where(ok, slots, 0)].reshape(n, -1)).to(dt)
        got = out.cpu()
        assert bool((got[~ok] == 7).all()) and bool((got[:, hkv * d:] == 7).all())
        assert torch.equal(got[ok, :hkv * d].isnan(), want[ok].isnan())
        assert torch.equal(got[ok, :hkv * d].nan_to_num(), want[ok].nan_to_num())
    # fewer pages than the tensors hold
    one = torch.full((n, hkv * d), 7.0, dtype=dt, device="cuda")
    luc.kv8_read(one, one.clone(), dev, k, v, scales, 1, 2, hkv, d, num_blocks=4)
    assert bool((one.cpu()[slots >= 4 * PAGE] == 7).all())


def test_another_stream_and_a_captured_append(luc):
    """Replays of a captured append of the same page, louder every time, against eager ones."""
    books = [Book(luc, 14, 2, 64, "bf16", seed=5) for _ in range(2)]
    a, b = 14 * 64, 16 * 64
    q_in = books[0].rows(3)
    slots = torch.tensor([17, 18, 5 * PAGE], device="cuda")
    pos = torch.tensor([1, 2, 80], dtype=torch.int32, device="cuda")
    q_out = torch.zeros(3, a, dtype=torch.bfloat16, device="cuda")

    def call(book, qkv, out, stream=None):
        luc.kv8_append(qkv[:, :a], qkv[:, a:b], qkv[:, b:], book.cos, book.sin, pos, slots, book.k, book.v, book.scales, 1, 2,
                       14, 2, 64, bounds=book.bounds, q_out=out, stream=stream, **books[0].kw)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(books[0], q_in, q_out)
    stream = torch.cuda.Stream()
    for i in range(5):
        q_in.copy_(books[0].rows(3, 3.0 ** i, 2.0 ** i))
        graph.replay()
        other = torch.zeros_like(q_out)
        stream.wait_stream(torch.cuda.current_stream())
        call(books[1], q_in, other, stream)
        torch.cuda.synchronize()
        assert torch.equal(q_out, other)
        for name in ("k", "v", "scales", "bounds"):
            x, y = getattr(books[0], name), getattr(books[1], name)
            assert torch.equal(x, y), name
