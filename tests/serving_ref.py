"""Plain 64-bit forms of the page maps, the normed appends and the 4-bit cache, for the tests.

Written from the formulas (include/luc_attn.h): per token and per head, no packed arithmetic."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE, GROUP, LIMIT = 16, 32, 60000.0


# ---- page maps ----------------------------------------------------------------------------

class Maps:
    """One sequence and one page at a time."""

    def __init__(self, batch, stride, num_blocks):
        self.lens = [0] * batch
        self.tables = np.zeros((batch, stride), np.int32)
        self.free = list(range(num_blocks - 1, -1, -1))

    def extend(self, new):
        slots, positions, cu, start = [], [], [0], list(self.lens)
        for b, n in enumerate(new):
            for _ in range(n):
                pos = self.lens[b]
                if pos % PAGE == 0:
                    self.tables[b, pos // PAGE] = self.free.pop()
                slots.append(int(self.tables[b, pos // PAGE]) * PAGE + pos % PAGE)
                positions.append(pos)
                self.lens[b] += 1
            cu.append(len(slots))
        return slots, positions, cu, start

    def truncate(self, keep):
        for b in reversed(range(len(keep))):
            want = min(keep[b], self.lens[b])
            for page in reversed(range(-(-want // PAGE), -(-self.lens[b] // PAGE))):
                self.free.append(int(self.tables[b, page]))
                self.tables[b, page] = 0
            self.lens[b] = want


# ---- the 4-bit format, f32 arithmetic as it is defined --------------------------------------

def encode(x):
    """x float32 array [..., d] of 16-bit values: (n uint8 [..., d], s, m fp16 [..., d / 32])."""
    with np.errstate(invalid="ignore", over="ignore"):
        g = np.clip(x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP).astype(np.float32), np.float32(-LIMIT), np.float32(LIMIT))
        nan = np.isnan(g).any(-1)
        m = g.min(-1).astype(np.float16)
        s = np.maximum((g.max(-1) - m.astype(np.float32)) / np.float32(15), np.float32(0)).astype(np.float16)
        sf = s.astype(np.float32)[..., None]
        q = np.where(sf > 0, (g - m.astype(np.float32)[..., None]) / np.where(sf > 0, sf, np.float32(1)), np.float32(0))
        n = np.clip(np.rint(q), 0, 15)
    n[nan] = 0
    s[nan] = m[nan] = np.float16(np.nan)
    return n.reshape(x.shape).astype(np.uint8), s, m


def values(n, s, m):
    """float64 values of n [..., d] with s, m [..., d / 32]."""
    g = n.reshape(*n.shape[:-1], n.shape[-1] // GROUP, GROUP).astype(np.float64)
    return (g * s.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]).reshape(n.shape)


def k_bytes(n, s, m, slab, t):
    """Writes token t (of 16) of one head into a K slab (uint8 [10 d])."""
    d = n.shape[-1]
    for x in range(0, d, 2):
        slab[t * (d // 2) + x // 2] = n[x] | n[x + 1] << 4
    sm = slab[8 * d:].view(np.float16)
    for g in range(d // GROUP):
        sm[(t * (d // GROUP) + g) * 2] = s[g]
        sm[(t * (d // GROUP) + g) * 2 + 1] = m[g]


def v_bytes(n, s, m, slab, t):
    d = n.shape[-1]
    o, i = t // 8, t % 8
    for x in range(0, d, 4):
        at = (o * (d // 4) + x // 4) * 16 + i * 2
        slab[at] = n[x] | n[x + 1] << 4
        slab[at + 1] = n[x + 2] | n[x + 3] << 4
    sm = slab[8 * d:].view(np.float16)
    for g in range(d // GROUP):
        sm[(o * (d // GROUP) + g) * 16 + i] = s[g]
        sm[(o * (d // GROUP) + g) * 16 + 8 + i] = m[g]


def pack_pool(x, is_v):
    """A pool of slabs [..., 10 d] from values x [..., 16, d] (float32), and the float64 values."""
    n, s, m = encode(x)
    lead, d = x.shape[:-2], x.shape[-1]
    by = n[..., 0::2] | n[..., 1::2] << 4
    if is_v:
        by = by.reshape(*lead, 2, 8, d // 4, 2).swapaxes(-3, -2)
        sm = np.stack([s, m], -1).reshape(*lead, 2, 8, d // GROUP, 2)
        sm = np.moveaxis(sm, -3, -1)
    else:
        sm = np.stack([s, m], -1)
    sm = np.ascontiguousarray(sm).view(np.uint8)
    pool = np.concatenate([by.reshape(*lead, 8 * d), sm.reshape(*lead, 2 * d)], -1)
    return pool, values(n, s, m)


# ---- norm, rotation -----------------------------------------------------------------------

def norm_rope(x, bias, norm, eps, cos, sin):
    """float64 heads x [rows, heads, d] (bias [heads, d]): (result, the size of its terms)."""
    x = x.double()
    if bias is not None:
        x = x + bias.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return (torch.cat([a * c - b * s, a * s + b * c], -1),
            torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1))


def append_tolerance(want, terms, dtype):
    """One rounding to dtype (half a step, and of the smallest subnormals), and f32 arithmetic before
    it: the bias, the sum of squares (16 in a chain, 3 more adds: 20 roundings, half of that on
    its root), mean, root, reciprocal, two products of the norm, a product and the sum of the rotation: fewer
    than 20 roundings of 2^-24, each relative to the terms."""
    fi = torch.finfo(dtype)
    return fi.eps / 2 * want.abs() * (1 + 1e-3) + fi.smallest_normal * fi.eps + 20 * 2.0 ** -24 * terms


# ---- attention ----------------------------------------------------------------------------

def attention(q, k, v, start, scale):
    """Rows q [n, hq, d] at positions start on over k, v [ctx, hkv, d] (float64): (out, tolerance
    without the output's own rounding).

    The kernels take k, v and q's products in fp16 operands with f32 sums.  Each value of K and V
    is off by up to half a step of fp16, 2^-11 of itself, spread evenly: 2^-11 / sqrt(3) in the
    mean square.  A score is then off by d_t = scale * 2^-11 / sqrt(3) * sqrt(sum (q k)^2), a
    weight by that and its own truncation to fp16 (within 2^-11 of its mean, which the sum of
    the truncated weights shares).  The roundings are independent, so their sum over the
    tokens grows as the root of the squares; six times it is taken.  Weights below 2^-14 of the
    largest lose up to 2^-24 each, and f32 sums of T terms up to T 2^-24 of the sum of their sizes.

    Where n and m are multiplied apart, n's weight is w s in two fp16 parts.  The second part (the
    remainder of the first, below 2^-10 of it) is mostly subnormal, a multiple of 2^-24, and two
    roundings to that take up to 2^-25 each: 2^-24 n <= 15 * 2^-24 a token, also where v = n s + m
    itself is near 0.  The weights' largest is at least 1, so of the output this is p_max times
    as much, T tokens at most, or six times sqrt(T / 3) where they are many."""
    n, hq, d = q.shape
    ctx, hkv = k.shape[:2]
    g = hq // hkv
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.empty_like(out)
    at = torch.arange(ctx, device=q.device)[None]
    limit = (start + torch.arange(n, device=q.device))[:, None]
    half = 2.0 ** -11
    for j in range(hq):
        kj, vj = k[:, j // g], v[:, j // g]
        kt = kj.t().contiguous()
        s = (q[:, j] @ kt) * scale
        s = torch.where(at <= limit, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, -1)
        o = p @ vj
        dt2 = (q[:, j] ** 2 @ (kt ** 2)) * (scale * half) ** 2 / 3 + half ** 2
        w2 = p * p * dt2
        # sum_t w2 (v - o)^2 = sum w2 v^2 - 2 o sum w2 v + o^2 sum w2
        spread = (w2 @ vj ** 2) - 2 * o * (w2 @ vj) + o * o * w2.sum(-1, keepdim=True)
        own = (p * p) @ vj ** 2 * half ** 2 / 3
        out[:, j] = o
        tol[:, j] = 6 * torch.sqrt((spread + own).clamp(min=0)) + \
            ctx * 2.0 ** -24 * vj.abs().amax() + 2.0 ** -20 * (p @ vj.abs()) + \
            p.amax(-1, keepdim=True) * min(ctx, 6 * math.sqrt(ctx / 3)) * 15 * 2.0 ** -24
    return out, tol


def check(got, want, tol, dtype, what):
    fi = torch.finfo(dtype)
    tol = tol + fi.eps / 2 * (want.abs() + tol) + fi.smallest_normal * fi.eps
    err = (got.double() - want).abs()
    worst = float((err / tol).max()) if err.numel() else 0.0
    print(f"  {what}: max error {float(err.max()) if err.numel() else 0.0:.3e}, {worst:.3f} of its tolerance", flush=True)
    assert torch.isfinite(got).all(), what
    assert worst <= 1.0, (what, worst)
