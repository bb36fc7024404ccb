"""Plain forms of the 8-bit cache for the tests, from the formulas (include/luc_attn.h): per page and per
head, in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE, LIMIT, LEAST = 16, 60000.0, -64


def _table():
    """The 256 e4m3 values, from their bits."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out[b] = math.nan if b & 127 == 127 else -x if b >> 7 else x
    return out


TABLE = _table()
_POSITIVE = TABLE[:127]  # 0 .. 448, ascending with the code


def encode(x):
    """The codes of float64 x (|x| <= 448 or NaN): the nearest, ties to the even code."""
    a = np.abs(x)
    nan = np.isnan(a)
    a = np.where(nan, 0.0, a)
    assert (a <= 448).all()
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    to_lo, to_hi = a - _POSITIVE[lo], _POSITIVE[hi] - a
    code = np.where((to_lo < to_hi) | ((to_lo == to_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(nan, 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def exponent(amax, most=448.0):
    """The smallest e >= LEAST with amax <= most * 2^e."""
    e = LEAST
    while amax > math.ldexp(most, e):
        e += 1
    return e


def exponents(x, most=448.0):
    """exponent() of every element of a float64 array."""
    m, e = np.frexp(np.asarray(x) / most)  # x / most = m 2^e with m in [1/2, 1): at most 2^e, 2^(e - 1) where m is 1/2
    return np.maximum(np.where(x > 0, e - (m == 0.5), LEAST), LEAST).astype(np.int64)


def k_slab(codes):
    """Bytes [16 d] of codes [16, d]."""
    return codes.reshape(-1)


def v_slab(codes):
    d = codes.shape[1]
    out = np.empty(16 * d, np.uint8)
    for t in range(16):
        for i in range(d):
            out[(t // 4 * d + i) * 4 + t % 4] = codes[t, i]
    return out


def of_slab(slab, is_v):
    """Codes [16, d] of bytes [16 d]."""
    d = slab.size // 16
    if not is_v:
        return slab.reshape(16, d)
    t, i = np.meshgrid(np.arange(16), np.arange(d), indexing="ij")
    return slab[(t // 4 * d + i) * 4 + t % 4]


class Pools:
    """8-bit pools on the host: [pages, layers, hkv, ...]."""

    def __init__(self, pages, layers, hkv, d, fill=0, scale=1.0):
        self.d = d
        self.k = np.full((pages, layers, hkv, 16 * d), fill, np.uint8)
        self.v = self.k.copy()
        self.scales = np.full((pages, layers, hkv, 2), scale, np.float32)
        self.bounds = np.full((pages, layers, hkv, 2, d), fill, np.uint8)

    def device(self):
        return [torch.from_numpy(x.copy()).cuda() for x in (self.k, self.v, self.scales, self.bounds)]

    def append(self, layer, slots, k, v):
        """Rows k, v float64 [rows, hkv, d] (16-bit values) to slots, those of a page at once."""
        runs = {}
        for r, s in enumerate(slots):
            if 0 <= s < self.k.shape[0] * PAGE:
                runs.setdefault(int(s) // PAGE, []).append((int(s) % PAGE, r))
        for page, rows in runs.items():
            offs = [o for o, _ in rows]
            joins = 0 not in offs
            at = [r for _, r in rows]
            for h in range(k.shape[1]):
                for is_v, x, pool in ((0, k, self.k), (1, v, self.v)):
                    x = x[at, h]
                    x = np.where(np.isnan(x), x, np.clip(x, -LIMIT, LIMIT))
                    e = exponent(float(np.abs(np.nan_to_num(x)).max()))
                    codes = of_slab(pool[page, layer, h], is_v).copy()
                    less = 0
                    if joins:
                        held = max(int(math.frexp(self.scales[page, layer, h, is_v])[1]) - 1, LEAST)
                        e = max(e, held)
                        less = held - e
                    if less:
                        codes = encode(TABLE[codes] * 2.0 ** less)
                    new = encode(x * 2.0 ** -e)
                    codes[offs] = new
                    pool[page, layer, h] = v_slab(codes) if is_v else k_slab(codes)
                    self.scales[page, layer, h, is_v] = 2.0 ** e
                    if is_v:
                        continue
                    y = np.nan_to_num(TABLE[new])
                    b = self.bounds[page, layer, h]
                    if joins:
                        old = np.nan_to_num(TABLE[encode(TABLE[b] * 2.0 ** less)])
                        y = np.concatenate([y, old])
                    b[0], b[1] = encode(y.max(0)), encode(y.min(0))

    def values(self, page_ids, layer, is_v):
        """float64 [16 pages, hkv, d] that pages hold."""
        pool = self.v if is_v else self.k
        out = [np.stack([TABLE[of_slab(pool[p, layer, h], is_v)] * float(self.scales[p, layer, h, int(is_v)])
                         for h in range(pool.shape[2])], 1) for p in page_ids]
        return np.concatenate(out) if out else np.empty((0, pool.shape[2], self.d))


def equal_codes(a, b):
    """Bytes that are the same codes (0 and -0, and all NaN, are one)."""
    x, y = TABLE[a], TABLE[b]
    return bool(((x == y) | (np.isnan(x) & np.isnan(y))).all())


# ---- attention ----------------------------------------------------------------------------

def attention(q, k, v, seen, scale, dtype):
    """Rows q [n, hq, d] over k, v [tokens, hkv, d] (float64; row r sees where seen [n, tokens]): (out, tolerance
    without the output's own rounding).

    K, V and q enter the products as they are, in dtype; the sums are f32.  A weight is rounded to dtype, by at
    most half a step, u = eps / 2 of itself, evenly spread (u / sqrt(3) in the mean square), and the weights' sum is that of the
    rounded ones: the output moves by sum_t p_t r_t (v_t - o), roundings independent, six times the root of the
    squares' sum is taken (where few weights count, each error is below sqrt(3) of its own).  A score's sum of d
    products in f32 is off by at most d 2^-24 sum |q k|, its scaling by as much as 3 2^-24 of its size in powers of two (at most
    1.5 times that of the exponent); each moves the output by p_t (v_t - o) times itself.  f32 sums of T
    terms: up to T 2^-24 of the sum of sizes; the exponential, merges and the quotient 2^-20 of it."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.empty_like(out)
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    for j in range(hq):
        kt, vj = k[:, j // g].t().contiguous(), v[:, j // g]
        s = (q[:, j] @ kt) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, -1)
        o = p @ vj
        size = (q[:, j].abs() @ kt.abs()) * abs(scale)
        off = f * (d * size + 4.5 * torch.where(seen, s, torch.zeros_like(s)).abs())
        w2 = p * p * u * u / 3
        spread = (w2 @ vj ** 2) - 2 * o * (w2 @ vj) + o * o * w2.sum(-1, keepdim=True)
        po = p * off
        out[:, j] = o
        tol[:, j] = 6 * torch.sqrt(spread.clamp(min=0)) + po @ vj.abs() + po.sum(-1, keepdim=True) * o.abs() + \
            (k.shape[0] * f + 2.0 ** -20) * (p @ vj.abs())
    return out, tol


# ---- the choice of pages --------------------------------------------------------------------

def scores(q, bounds, scale):
    """float32 scores [pages] of one kv head: q float64 [group, d], bounds codes [pages, 2, d], scale float32 [pages]."""
    whole = np.rint(np.nan_to_num(TABLE[bounds]))
    best = np.full(len(bounds), -np.inf, np.float32)
    for x in q:
        x = np.clip(np.nan_to_num(x, posinf=LIMIT, neginf=-LIMIT), -LIMIT, LIMIT)
        total = np.zeros(len(bounds), np.float32)
        for j in range(0, x.size, 32):
            e = exponent(float(np.abs(x[j:j + 32]).max()), 127.0)
            n = np.rint(x[j:j + 32] * 2.0 ** -e)
            s = (np.where(n > 0, whole[:, 0, j:j + 32], whole[:, 1, j:j + 32]) * n).sum(-1)
            total = total + (s * 2.0 ** e).astype(np.float32)
        best = np.maximum(best, total)
    return best * scale


def choose(score, budget, first, recent, bad=()):
    """The chosen of len(score) pages, ascending, -1 behind the last."""
    count = len(score)
    if count <= budget:
        return list(range(count)) + [-1] * (budget - count)
    rank = [(math.inf if p < first or p >= count - recent else -math.inf if p in bad else float(score[p]), -p)
            for p in range(count)]
    return sorted(sorted(range(count), key=lambda p: rank[p], reverse=True)[:budget])
