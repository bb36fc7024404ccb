"""luc_qk_norm_rope_append and luc_kv4_append against 64-bit results, the older append and the
4-bit format written byte by byte."""
import numpy as np
import pytest
import torch

import serving_ref as ref
from gpu_util import from_dev

pytestmark = pytest.mark.gpu
PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def rope(max_pos, d):
    i = np.arange(d // 2) * 2.0 / d
    th = np.arange(max_pos)[:, None] / 1e6 ** i[None]
    return (torch.from_numpy(np.cos(th).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(th).astype(np.float32)).cuda())


class Case:
    def __init__(self, rows, hq, hkv, d, dtype, norm, bias, seed=0, layers=2, extra=0, scale=1.4):
        gen = torch.Generator().manual_seed(seed)
        dt = DT[dtype]
        self.rows, self.hq, self.hkv, self.d, self.dt, self.layers = rows, hq, hkv, d, dt, layers
        width = (hq + 2 * hkv) * d
        rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.buf = (rnd(rows, width + extra) * scale).to(dt).cuda()
        self.qkv = self.buf[:, :width]
        self.bias = (rnd(width) * 0.3).to(dt).cuda() if bias else None
        self.q_norm = (1 + 0.2 * rnd(d)).to(dt).cuda() if norm else None
        self.k_norm = (1 + 0.2 * rnd(d)).to(dt).cuda() if norm else None
        rng = np.random.default_rng(seed)
        self.pages = rows // PAGE + 3
        self.slots = torch.from_numpy(rng.permutation(self.pages * PAGE)[:rows].astype(np.int64)).cuda()
        self.pos = torch.from_numpy(rng.integers(0, 900, rows).astype(np.int32)).cuda()
        self.cos, self.sin = rope(900, d)

    def views(self):
        a, b = self.hq * self.d, (self.hq + self.hkv) * self.d
        return self.qkv[:, :a], self.qkv[:, a:b], self.qkv[:, b:]

    def kw(self):
        a, b = self.hq * self.d, (self.hq + self.hkv) * self.d
        kw = dict(q_norm=self.q_norm, k_norm=self.k_norm, eps=1e-6)
        if self.bias is not None:
            kw.update(q_bias=self.bias[:a], k_bias=self.bias[a:b], v_bias=self.bias[b:])
        return kw

    def pools(self, four, fill=0):
        shape = (self.pages, self.layers, self.hkv, 10 * self.d) if four else \
            (self.pages, self.layers, self.hkv, PAGE, self.d)
        return [torch.full(shape, fill, dtype=torch.uint8 if four else self.dt, device="cuda") for _ in range(2)]

    def run(self, luc, four, q_out=None, outs=(None, None), pools=None, layer=1, stream=None, slots=None,
            pos=None, num_blocks=None):
        kp, vp = pools or self.pools(four)
        q, k, v = self.views()
        kw = self.kw() | dict(q_out=q_out, k_out=outs[0], stream=stream, num_blocks=num_blocks)
        if four:
            kw["v_out"] = outs[1]
        print(f"  append{4 if four else 16}: {self.rows} rows {self.hq}/{self.hkv}x{self.d} {self.dt}", flush=True)
        (luc.kv4_append if four else luc.qk_norm_rope_append)(
            q, k, v, self.cos, self.sin, self.pos if pos is None else pos,
            self.slots if slots is None else slots, kp, vp, layer, self.layers, self.hq, self.hkv, self.d, **kw)
        torch.cuda.synchronize()
        return kp, vp

    def exact(self):
        q, k, v = (t.reshape(self.rows, -1, self.d) for t in self.views())
        kw = self.kw()
        head = lambda b: None if b is None else b.view(-1, self.d)  # noqa: E731
        c, s = self.cos[self.pos.long()], self.sin[self.pos.long()]
        vv = v.double() if self.bias is None else v.double() + head(kw["v_bias"]).double()
        return (ref.norm_rope(q, head(kw.get("q_bias")), self.q_norm, 1e-6, c, s),
                ref.norm_rope(k, head(kw.get("k_bias")), self.k_norm, 1e-6, c, s), (vv, vv.abs()))

    def at_slots(self, pool, layer=1):
        return pool[self.slots // PAGE, layer, :, self.slots % PAGE]


SIZES = [(1, 14, 2, 64), (2, 4, 4, 128), (5, 28, 4, 128), (17, 8, 8, 64), (100, 12, 2, 128), (333, 14, 2, 64),
         (64, 32, 8, 128), (31, 8, 1, 64)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm,bias", [(True, False), (True, True), (False, True), (False, False)])
@pytest.mark.parametrize("rows,hq,hkv,d", SIZES)
def test_16_bit_against_64_bit_results(luc, rows, hq, hkv, d, norm, bias, dtype):
    c = Case(rows, hq, hkv, d, dtype, norm, bias, seed=rows)
    q_out = torch.full((rows, hq * d), 7.0, dtype=c.dt, device="cuda")
    k_out = torch.full((rows, hkv * d), 7.0, dtype=c.dt, device="cuda")
    before = c.buf.clone()
    kp, vp = c.run(luc, False, q_out, (k_out, None))
    assert torch.equal(c.buf, before)
    (q, qt), (k, kt), (v, vt) = c.exact()
    for got, want, terms in ((q_out.view(rows, hq, d), q, qt), (k_out.view(rows, hkv, d), k, kt),
                             (c.at_slots(vp), v, vt)):
        tol = ref.append_tolerance(want, terms, c.dt)
        assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(c.at_slots(kp), k_out.view(rows, hkv, d))
    # nothing else: the other layer, the other slots
    for p in (kp, vp):
        assert not p[:, 0].any()
        p[c.slots // PAGE, 1, :, c.slots % PAGE] = 0
        assert not p.any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("rows,hq,hkv,d", SIZES[:6])
def test_without_norms_the_bits_of_rope_append(luc, rows, hq, hkv, d, bias, dtype):
    c = Case(rows, hq, hkv, d, dtype, False, bias, seed=rows + 1, layers=1)
    # luc_rope_append's slots: table row r is row r, its page where the position falls
    tables = torch.zeros((rows, 900 // PAGE + 1), dtype=torch.int32, device="cuda")
    perm = torch.randperm(rows).int().cuda()
    tables[torch.arange(rows, device="cuda"), (c.pos // PAGE).long()] = perm
    c.pages = rows
    c.slots = perm.long() * PAGE + c.pos % PAGE
    qkv = c.qkv.clone()
    kp0, vp0 = c.pools(False)
    a, b = hq * d, (hq + hkv) * d
    kw = c.kw()
    luc.rope_append(qkv, kw.get("q_bias"), qkv[:, a:], kw.get("k_bias"), qkv[:, b:], kw.get("v_bias"),
                    qkv.shape[1], c.cos, c.sin, c.pos, tables, kp0, vp0, rows, 0, 1, hq, hkv, d)
    kp, vp = c.run(luc, False, outs=(c.views()[1], None), layer=0)  # in place
    for x, y in ((c.qkv, qkv), (kp, kp0), (vp, vp0)):
        assert np.array_equal(from_dev(x), from_dev(y))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm,bias", [(True, False), (False, True)])
@pytest.mark.parametrize("rows,hq,hkv,d", SIZES)
def test_4_bit_pool_byte_by_byte(luc, rows, hq, hkv, d, norm, bias, dtype):
    """The pool's bytes are those of the format for the 16-bit values that the other append
    writes; q is the same; k_out and v_out are the format's values."""
    c = Case(rows, hq, hkv, d, dtype, norm, bias, seed=2 * rows, extra=24)
    q0, q1 = (torch.zeros((rows, hq * d), dtype=c.dt, device="cuda") for _ in range(2))
    kp16, vp16 = c.run(luc, False, q0)
    outs = [torch.zeros((rows, hkv * d), dtype=c.dt, device="cuda") for _ in range(2)]
    kp, vp = c.run(luc, True, q1, outs, pools=c.pools(True, 0xAB))
    assert torch.equal(q0, q1)
    slots = c.slots.tolist()
    for pool, src, write, out in ((kp, kp16, ref.k_bytes, outs[0]), (vp, vp16, ref.v_bytes, outs[1])):
        x = c.at_slots(src).float().cpu().numpy()  # [rows, hkv, d]
        n, s, m = ref.encode(x)
        want = np.full(tuple(pool.shape), 0xAB, np.uint8)
        for r, slot in enumerate(slots):
            for h in range(hkv):
                write(n[r, h], s[r, h], m[r, h], want[slot // PAGE, 1, h], slot % PAGE)
        assert np.array_equal(pool.cpu().numpy(), want)
        val = torch.from_numpy(ref.values(n, s, m)).float().to(c.dt)
        assert torch.equal(out.cpu().view(rows, hkv, d), val)
        # half a step of the group, s / 2, and the roundings of m and s to fp16
        step = np.repeat(s.astype(np.float64), 32, -1)
        size = np.abs(x).max()
        assert (np.abs(ref.values(n, s, m) - x) <= step / 2 + 2.0 ** -10 * size).all()


def test_4_bit_of_unusual_values(luc):
    """Constant groups, subnormals, values past the limit, infinities and NaN, as the format says."""
    c = Case(8, 2, 2, 64, "bf16", False, False, seed=5)
    x = c.qkv.view(8, 6, 64)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = 1e-7
    x[2, :, ::3] = -2e-7
    x[3, :, 5] = 1e30
    x[4, :, 7] = float("inf")
    x[4, :, 40] = float("-inf")
    x[5, :, 3] = float("nan")
    x[6] *= 1e4
    x[7] = -60000.0
    c.pos.zero_()  # no rotation: k is what goes in
    outs = [torch.zeros((8, 128), dtype=c.dt, device="cuda") for _ in range(2)]
    kp, vp = c.run(luc, True, torch.zeros((8, 128), dtype=c.dt, device="cuda"), outs)
    for pool, src, write, out in ((kp, x[:, 2:4], ref.k_bytes, outs[0]), (vp, x[:, 4:6], ref.v_bytes, outs[1])):
        v = src.float()
        if src.data_ptr() == x[:, 2:4].data_ptr():  # at position 0: x1 * 1 - x2 * 0 | x1 * 0 + x2 * 1
            a, b = v[..., :32], v[..., 32:]
            v = torch.cat([a * 1 - b * 0, a * 0 + b * 1], -1).to(c.dt).float()
        n, s, m = ref.encode(v.cpu().numpy())
        want = np.zeros(tuple(pool.shape), np.uint8)
        for r, slot in enumerate(c.slots.tolist()):
            for h in range(2):
                write(n[r, h], s[r, h], m[r, h], want[slot // PAGE, 1, h], slot % PAGE)
        got = pool.cpu().numpy()
        nan = lambda a: np.where(np.isnan(a), np.float16(9999), a)  # noqa: E731
        assert np.array_equal(got[..., :512], want[..., :512])
        assert np.array_equal(nan(got[..., 512:].view(np.float16)), nan(want[..., 512:].view(np.float16)))
        val = torch.from_numpy(ref.values(n, s, m)).float().to(c.dt)
        assert torch.equal(torch.nan_to_num(out.cpu().view(8, 2, 64), 9.0), torch.nan_to_num(val, 9.0))


@pytest.mark.parametrize("four", [False, True])
def test_rows_without_a_slot_or_position(luc, four):
    """Slots -1 and past the pool: q and k are formed, nothing is cached.  Positions outside the
    tables: nothing at all."""
    c = Case(40, 14, 2, 64, "f16", True, False, seed=9)
    q_all = torch.zeros((40, 14 * 64), dtype=c.dt, device="cuda")
    kp0, vp0 = c.run(luc, four, q_all)
    slots, pos = c.slots.clone(), c.pos.clone()
    nb = c.pages - 1
    slots[::4] = -1
    slots[1::8] = nb * PAGE
    slots[3::16] = 1 << 40
    pos[2::8] = -1
    pos[5::8] = 900
    q = torch.full_like(q_all, 7.0)
    outs = [torch.full((40, 128), 7.0, dtype=c.dt, device="cuda") for _ in range(2)]
    kp, vp = c.run(luc, four, q, outs, slots=slots, pos=pos, num_blocks=nb)
    gone = (pos < 0) | (pos >= 900)
    assert torch.equal(q[~gone], q_all[~gone]) and bool((q[gone] == 7).all())
    assert bool((outs[0][gone] == 7).all()) and bool((outs[0][~gone] != 7).any(-1).all())
    kept = ~gone & (slots >= 0) & (slots < nb * PAGE)
    c2 = c.slots[kept]
    if four:
        want_k, want_v = c.pools(True)
        sub = Case(40, 14, 2, 64, "f16", True, False, seed=9)
        keep_slots = torch.where(kept, slots, torch.full_like(slots, -1))
        sub.run(luc, True, torch.zeros_like(q_all), pools=(want_k, want_v), slots=keep_slots)
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
        assert bool((kp[c2 // PAGE, 1] != 0).any())
    else:
        want = torch.zeros_like(kp0)
        want[c2 // PAGE, 1, :, c2 % PAGE] = kp0[c2 // PAGE, 1, :, c2 % PAGE]
        assert torch.equal(kp, want)


def test_offsets_past_32_bits(luc):
    """The last page of pools of more than 4 GiB."""
    c = Case(16, 4, 4, 128, "bf16", True, False, seed=4, layers=1)
    small = torch.zeros((16, 4 * 128), dtype=c.dt, device="cuda")
    first = torch.arange(16, device="cuda")
    c.pages = 2
    kp, vp = c.run(luc, True, small, layer=0, slots=first + PAGE)
    kp16, _ = c.run(luc, False, small, layer=0, slots=first + PAGE)
    for four, src in ((True, kp), (False, kp16)):
        c.pages = (1 << 32) // (src[0].numel() * src.element_size()) + 5
        big, bigv = c.pools(four)
        c.run(luc, four, small, pools=(big, bigv), layer=0, slots=first + (c.pages - 1) * PAGE)
        assert torch.equal(big[-1], src[1]) and not big[:-1].view(torch.int64).any()
        del big, bigv
        torch.cuda.empty_cache()


def test_another_stream_and_a_captured_append(luc):
    c = Case(70, 28, 4, 128, "bf16", True, True, seed=6)
    q0, q1 = (torch.zeros((70, 28 * 128), dtype=c.dt, device="cuda") for _ in range(2))
    kp0, vp0 = c.run(luc, True, q0)
    kp1, vp1 = c.pools(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    c.run(luc, True, q1, pools=(kp1, vp1), stream=stream)
    assert torch.equal(q0, q1) and torch.equal(kp0, kp1) and torch.equal(vp0, vp1)
    graph = torch.cuda.CUDAGraph()
    q, k, v = c.views()
    with torch.cuda.graph(graph):
        luc.kv4_append(q, k, v, c.cos, c.sin, c.pos, c.slots, kp1, vp1, 1, c.layers, c.hq, c.hkv, c.d,
                       q_out=q1, **c.kw())
    for seed in range(3):
        other = Case(70, 28, 4, 128, "bf16", True, True, seed=6)
        other.qkv.copy_(torch.randn(other.qkv.shape, generator=torch.Generator().manual_seed(seed)))
        c.qkv.copy_(other.qkv)
        graph.replay()
        kp2, vp2 = other.run(luc, True, q0)
        assert torch.equal(q0, q1) and torch.equal(kp2, kp1) and torch.equal(vp2, vp1)


@pytest.mark.parametrize("four", [False, True])
def test_one_row_of_tensors_of_their_own(luc, four):
    """A single token's q, k and v in three tensors: the row of a shared qkv tensor."""
    c = Case(1, 14, 2, 64, "f16", True, True)
    want = torch.empty(1, 14 * 64, dtype=c.dt, device="cuda")
    pools = c.pools(four)
    c.run(luc, four, q_out=want, pools=pools)
    q, k, v = (x.clone() for x in c.views())
    got, again = torch.empty_like(want), c.pools(four)
    call = luc.kv4_append if four else luc.qk_norm_rope_append
    call(q, k, v, c.cos, c.sin, c.pos, c.slots, *again, 1, c.layers, 14, 2, 64, q_out=got, **c.kw())
    assert torch.equal(got, want)
    for a, b in zip(pools, again):
        assert torch.equal(a, b)
