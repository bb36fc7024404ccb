"""Serving over a paged cache held in 8 bits, operator by operator: what is called, on what, and its plain form.

- "append": RMS norms of q's and k's heads, their rotation, and k and v into the 8-bit pool by
  slot, with each page's scales and key bounds brought up to date (`LucAttn.kv8_append`).
- "read": tokens of the pool back in 16 bits (`LucAttn.kv8_read`).
- "attn": attention of a batch's new rows over the pool (`LucAttn.kv8_attention`), one row a
  sequence (decode steps) or packed prompts.
- "sparse": for one row a sequence, the pages of its context that a score over the key bounds
  puts first, and attention over those alone (`LucAttn.kv8_select`,
  `LucAttn.kv8_sparse_attention`).

`own` chooses between the framework's calls and plain torch in `run`.  Pools hold, for each page of
16 tokens, layer and kv head, 16 * d e4m3 codes: K as [16 tokens][d], V as [4][d][4 tokens].  A
value is code * scale; scales [pages][layers][kv heads][K, V] in fp32 are powers of two, the smallest
that brings the page's largest value to at most 448, 2^-64 at least, and grow as rows arrive (the codes
that the page holds are rounded again then).  A page begins anew with its first token.  Key bounds,
[pages][layers][kv heads][largest, smallest][d], are codes too, of the page's own.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
EPS = 1e-6
ROPE_BASE = 1e6
LIMIT = 60000.0  # values beyond it are stored as it
LEAST = -64      # exponent of the smallest scale
FIRST, RECENT = 1, 2  # pages that every selection holds: the first, and the last two
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # the new rows of a serving batch (the benchmark's decode workload)
        {"name": "append_b32", "kind": "append", "rows": 32, "seqs": 32, "hq": 14, "hkv": 2,
         "d": 64, "dtype": "f16", "norm": False, "bias": True},
        # four long prompts, with head norms
        {"name": "append_prompts", "kind": "append", "rows": 8191, "seqs": 4, "hq": 28,
         "hkv": 4, "d": 128, "dtype": "bf16", "norm": True, "bias": False},
        # a short cached prefix, for a path that takes 16 bits
        {"name": "read_prefix", "kind": "read", "rows": 333, "hkv": 2, "d": 64, "dtype": "f16"},
        # a long document's tokens of one layer
        {"name": "read_document", "kind": "read", "rows": 32701, "hkv": 4, "d": 128, "dtype": "bf16"},
        # one sequence, short context: the latency of a chat's next token
        {"name": "attn_single", "kind": "attn", "batch": 1, "lo": 512, "hi": 512, "rows_lo": 1,
         "rows_hi": 1, "hq": 14, "hkv": 2, "d": 64, "dtype": "f16"},
        # a serving batch of mixed contexts (the benchmark's decode workload)
        {"name": "attn_b32_mixed", "kind": "attn", "batch": 32, "lo": 128, "hi": 4096,
         "rows_lo": 1, "rows_hi": 1, "hq": 14, "hkv": 2, "d": 64, "dtype": "f16"},
        # the largest decode: a full batch of long mixed contexts
        {"name": "attn_b64_long", "kind": "attn", "batch": 64, "lo": 1024, "hi": 16384,
         "rows_lo": 1, "rows_hi": 1, "hq": 28, "hkv": 4, "d": 128, "dtype": "bf16"},
        # a chunk of a long prompt after its cached prefix
        {"name": "attn_chunk", "kind": "attn", "batch": 1, "lo": 8000, "hi": 8000,
         "rows_lo": 512, "rows_hi": 512, "hq": 12, "hkv": 2, "d": 128, "dtype": "f16"},
        # long prompts of odd lengths from an empty cache
        {"name": "attn_prompts", "kind": "attn", "batch": 4, "lo": 0, "hi": 0, "rows_lo": 1531,
         "rows_hi": 2048, "hq": 14, "hkv": 2, "d": 64, "dtype": "bf16"},
        # one long document, the next token from 2048 of its tokens
        {"name": "sparse_single", "kind": "sparse", "batch": 1, "lo": 32768, "hi": 32768,
         "budget": 128, "hq": 12, "hkv": 2, "d": 128, "dtype": "bf16"},
        # a serving batch of mixed contexts, some shorter than the selection
        {"name": "sparse_b32_mixed", "kind": "sparse", "batch": 32, "lo": 128, "hi": 4096,
         "budget": 64, "hq": 14, "hkv": 2, "d": 64, "dtype": "f16"},
        # a full batch of long mixed contexts
        {"name": "sparse_b64_long", "kind": "sparse", "batch": 64, "lo": 1024, "hi": 16384,
         "budget": 96, "hq": 28, "hkv": 4, "d": 128, "dtype": "bf16"},
    ]


# head layouts in use: (query heads, kv heads, head_dim)
_HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 8, 64), (32, 8, 128), (4, 2, 64),
          (8, 8, 128), (16, 2, 128)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append"] * 2 + ["read"] + ["attn"] * 4 + ["sparse"] * 3)
    hq, hkv, d = rng.choice(_HEADS)
    dtype = rng.choice(["f16", "bf16"])
    if kind == "append":
        rows = _log_int(rng, 1, 8191 * 28 * 128 // (hq * d) if hq * d > 3584 else 8191)
        return {"kind": kind, "rows": rows, "seqs": min(rows, rng.choice([1, 3, 8, 64])),
                "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "norm": rng.choice([True, True, False]),
                "bias": rng.choice([True, False])}
    if kind == "read":
        return {"kind": kind, "rows": _log_int(rng, 1, 32701 * 512 // max(512, hkv * d)), "hkv": hkv, "d": d,
                "dtype": dtype}
    # at most 0.5 M tokens x heads x dimensions of 128
    most = 64 * 8700 * 4 * 128 // (hkv * d)
    if kind == "sparse":
        hi = _log_int(rng, 1, 65536)
        batch = _log_int(rng, 1, max(1, min(64, most // hi)))
        return {"kind": kind, "batch": batch, "lo": rng.choice([hi, max(1, hi // 2), max(1, hi // 16)]),
                "hi": hi, "budget": _log_int(rng, 8, 256), "hq": hq, "hkv": hkv, "d": d, "dtype": dtype}
    if rng.random() < 0.55:  # decode steps
        hi = _log_int(rng, 1, 32768)
        batch = _log_int(rng, 1, max(1, min(64, most // hi)))
        return {"kind": kind, "batch": batch, "lo": rng.choice([hi, max(1, hi // 2), max(1, hi // 16)]),
                "hi": hi, "rows_lo": 1, "rows_hi": 1, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype}
    batch = rng.choice([1, 1, 2, 3, 5, 8])
    hi = rng.choice([0, 0, _log_int(rng, 16, 12000)])
    rows = _log_int(rng, 2, 2048)
    # at most the listed prompts' products
    while 4.0 * d * hq * batch * rows * (hi + rows / 2 + 1) > 25e9:
        rows = max(2, rows * 3 // 4)
    return {"kind": kind, "batch": batch, "lo": hi // 3, "hi": hi,
            "rows_lo": rng.choice([rows, max(1, rows // 8)]), "rows_hi": rows,
            "hq": hq, "hkv": hkv, "d": d, "dtype": dtype}


# ---- inputs, from the seed alone; lengths belong to the case ------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(gen, shape, std, dtype, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean).to(dtype)


def _spread(lo, hi, n, salt):
    """n lengths between lo and hi, not sorted, the longest among them."""
    x = np.random.default_rng(n + salt).integers(lo, hi + 1, n)
    x[n // 2] = hi
    return x


def _lengths(case):
    """(cached tokens, new rows) of every sequence."""
    n = case["batch"]
    held = _spread(case["lo"], case["hi"], n, 0)
    if case["kind"] == "sparse" or case["rows_hi"] == 1:
        return held - 1, np.ones(n, np.int64)  # lo .. hi are the contexts, the new row's own token among them
    return held, _spread(case["rows_lo"], case["rows_hi"], n, 1000)


def _int32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _pages(tokens):
    return -(-np.asarray(tokens, dtype=np.int64) // PAGE)


def _deal(seed, total):
    """Tables with the pages of `total` tokens dealt from a shuffled pool: (tables, pages in the pool)."""
    tp = _pages(total)
    count = int(tp.sum() * 1.05) + 3
    perm = np.random.default_rng(int(seed)).permutation(count).astype(np.int32)
    tables = np.zeros((len(tp), max(1, int(tp.max()))), np.int32)
    starts = np.cumsum(tp) - tp
    for b in range(len(tp)):
        tables[b, :tp[b]] = perm[starts[b]:starts[b] + tp[b]]
    return tables, count


def _rope_table(n, d):
    """cos and sin [n][d / 2] in fp32, as the engine keeps them."""
    i = np.arange(d // 2, dtype=np.float32) * np.float32(2) / np.float32(d)
    freq = np.power(np.float32(ROPE_BASE), i, dtype=np.float32)
    theta = (np.arange(n, dtype=np.float32)[:, None] / freq[None]).astype(np.float64)
    return (torch.from_numpy(np.cos(theta).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(theta).astype(np.float32)).cuda())


# q and k of this size give scores of standard deviation about 2, as trained heads do
_QK_STD, _V_STD = 1.4, 1.0


def _pools(gen, pages, layers, hkv, d, bounds):
    """(k, v, scales, key bounds or None) as earlier appends filled them, in pieces.  The keys of a
    page are alike, as neighbouring tokens' are."""
    shape = (pages, layers, hkv)
    kp = torch.empty(shape + (PAGE * d,), dtype=torch.uint8, device="cuda")
    vp = torch.empty_like(kp)
    scales = torch.empty(shape + (2,), device="cuda")
    index = torch.empty(shape + (2, d), dtype=torch.uint8, device="cuda") if bounds else None
    step = max(1, (1 << 25) // (layers * hkv * PAGE * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        for is_v, pool in enumerate((kp, vp)):
            x = torch.randn((n, layers, hkv, PAGE, d), generator=gen, device="cuda")
            if is_v:
                x.mul_(_V_STD)
            else:
                x.add_(torch.randn((n, layers, hkv, 1, d), generator=gen, device="cuda")).mul_(_QK_STD / math.sqrt(2))
            e = _exponent(x.abs().amax((-1, -2)))
            scales[i:i + n, ..., is_v] = _pow2(e)
            codes = (x * _pow2(-e)[..., None, None]).to(_E4M3)
            pool[i:i + n] = _slab(codes, is_v).view(torch.uint8)
            if bounds and not is_v:
                f = codes.float()
                index[i:i + n] = torch.stack([f.amax(-2), f.amin(-2)], -2).to(_E4M3).view(torch.uint8)
    return kp, vp, scales, index


def prepare(case, seed):
    if case["kind"] == "append":
        return _prepare_append(case, seed)
    if case["kind"] == "read":
        return _prepare_read(case, seed)
    return _prepare_attn(case, seed)


def _prepare_append(case, seed):
    gen, dt = _gen(seed), _DT[case["dtype"]]
    hq, hkv, d, rows, seqs = case["hq"], case["hkv"], case["d"], case["rows"], case["seqs"]
    rng = np.random.default_rng(int(seed))
    new = np.full(seqs, rows // seqs)
    new[:rows % seqs] += 1
    # one row a sequence: a decode step, somewhere in its context; else prompts from the start
    start = rng.integers(0, 4000, seqs) if rows == seqs else np.zeros(seqs, np.int64)
    # pages for the new rows (and the page that a decode step's context ends in)
    first = start // PAGE
    counts = (start + new - 1) // PAGE - first + 1
    pages = rng.permutation(int(counts.sum()) + 2)
    base = np.cumsum(counts) - counts
    b = np.repeat(np.arange(seqs), new)
    pos = start[b] + np.arange(rows) - (np.cumsum(new) - new)[b]
    slots = pages[base[b] + pos // PAGE - first[b]] * PAGE + pos % PAGE
    cos, sin = _rope_table(int(pos.max()) + 1, d)
    kp, vp, scales, index = _pools(gen, len(pages), 1, hkv, d, True)  # (of earlier sequences, too)
    return {"case": case, "qkv": _normal(gen, (rows, (hq + 2 * hkv) * d), 1.4, dt), "cos": cos, "sin": sin,
            "positions": _int32(pos), "slots": torch.from_numpy(slots.astype(np.int64)).cuda(),
            "q_norm": _normal(gen, (d,), 0.1, dt, 1.0) if case["norm"] else None,
            "k_norm": _normal(gen, (d,), 0.1, dt, 1.0) if case["norm"] else None,
            "bias": _normal(gen, ((hq + 2 * hkv) * d,), 0.1, dt) if case["bias"] else None,
            "q_out": torch.zeros((rows, hq * d), dtype=dt, device="cuda"),
            "k_pool": kp, "v_pool": vp, "scales": scales, "index": index}


def _prepare_read(case, seed):
    gen, dt, rows = _gen(seed), _DT[case["dtype"]], case["rows"]
    hkv, d = case["hkv"], case["d"]
    tables, count = _deal(seed, [rows])
    kp, vp, scales, _ = _pools(gen, count, 1, hkv, d, False)
    pos = np.arange(rows)
    return {"case": case, "k_pool": kp, "v_pool": vp, "scales": scales,
            "slots": torch.from_numpy(tables[0, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE).cuda(),
            "k_out": torch.zeros((rows, hkv * d), dtype=dt, device="cuda"),
            "v_out": torch.zeros((rows, hkv * d), dtype=dt, device="cuda")}


def _prepare_attn(case, seed):
    gen, dt = _gen(seed), _DT[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    held, new = _lengths(case)
    tables, count = _deal(seed, held + new)
    cu = np.concatenate([[0], np.cumsum(new)])
    rows = int(cu[-1])
    q = _normal(gen, (rows, hq * d), _QK_STD, dt)
    kp, vp, scales, index = _pools(gen, count, 2, hkv, d, case["kind"] == "sparse")
    s = {"case": case, "q": q, "k_pool": kp, "v_pool": vp, "scales": scales, "index": index,
         "tables": _int32(tables), "cu": _int32(cu), "start": _int32(held),
         "max_ctx": int((held + new).max()), "max_rows": int(new.max()),
         "out": torch.zeros((rows, hq * d), dtype=dt, device="cuda")}
    if case["kind"] == "sparse":
        s["pages"] = torch.zeros((case["batch"], hkv, case["budget"]), dtype=torch.int32, device="cuda")
    return s


# ---- the 8-bit format in plain torch ------------------------------------------------------

def _pow2(e):
    """2^e in fp32, by its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(amax, most=1.75 * 256):
    """The smallest e with amax <= most * 2^e, exactly (amax fp32)."""
    m, e = torch.frexp(amax.clamp(max=LIMIT))
    top, shift = math.frexp(most)
    return torch.where(amax > 0, e - shift + (m > top), torch.full_like(e, LEAST)).clamp(min=LEAST)


def _slab(codes, is_v):
    """Codes [..., 16, d] in the order of a slab, flat."""
    if is_v:
        codes = codes.unflatten(-2, (4, 4)).transpose(-1, -2).contiguous()
    return codes.flatten(codes.dim() - (3 if is_v else 2))


def _values(slab, scale, is_v):
    """Values [..., 16, d] in fp32 of slabs [..., 16 d] and their scales."""
    d = slab.shape[-1] // PAGE
    x = slab.view(_E4M3).float()
    x = x.unflatten(-1, (4, d, 4)).transpose(-1, -2).flatten(-3, -2) if is_v else x.unflatten(-1, (PAGE, d))
    return x * scale[..., None, None]


# ---- one pass -----------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "append":
        return _append_own(state) if own else _append_plain(state)
    if kind == "read":
        return _read_own(state) if own else _read_plain(state)
    if kind == "attn":
        return _attn_own(state) if own else _attn_plain(state)
    return _sparse_own(state) if own else _sparse_plain(state)


def _append_outputs(s):
    return {"q": s["q_out"], "k": s["k_pool"].view(_E4M3), "v": s["v_pool"].view(_E4M3), "scales": s["scales"],
            "bounds": s["index"].view(_E4M3)}


def _append_plain(s):
    case = s["case"]
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], s["q_out"].dtype
    x = s["qkv"].float()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    x = x.unflatten(-1, (-1, d))
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    at = s["positions"].long()
    c, n = s["cos"][at][:, None], s["sin"][at][:, None]
    q1, q2 = q.chunk(2, -1)
    k1, k2 = k.chunk(2, -1)
    s["q_out"].copy_(torch.cat([q1 * c - q2 * n, q1 * n + q2 * c], -1).flatten(1))
    k = torch.cat([k1 * c - k2 * n, k1 * n + k2 * c], -1)
    page, off = s["slots"] // PAGE, s["slots"] % PAGE
    pages = s["k_pool"].shape[0]
    # the first of a page's offsets that are written: 0 begins it anew, 16 is a page of no row
    least = torch.full((pages,), PAGE, device="cuda", dtype=torch.int64).scatter_reduce(0, page, off, "amin")
    anew, here = (least == 0)[:, None], (least < PAGE)[:, None]
    for is_v, x, pool in ((0, k, s["k_pool"]), (1, v, s["v_pool"])):
        x = x.to(dt).float().clamp(-LIMIT, LIMIT)
        scale = s["scales"][:, 0, :, is_v]
        amax = torch.zeros((pages, hkv), device="cuda").scatter_reduce(
            0, page[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
        e, held = _exponent(amax), torch.frexp(scale)[1] - 1
        e = torch.where(here, torch.where(anew, e, torch.maximum(e, held)), held)
        less = torch.where(anew, torch.zeros_like(e), held - e)
        codes = _values(pool[:, 0], _pow2(less), is_v).to(_E4M3)
        new = (x * _pow2(-e)[page][..., None]).to(_E4M3)
        codes[page, :, off] = new
        pool[:, 0] = _slab(codes, is_v).view(torch.uint8)
        scale.copy_(_pow2(e))
        if not is_v:
            to = page[:, None, None].expand(-1, hkv, d)
            for side, reduce, none in ((0, "amax", -math.inf), (1, "amin", math.inf)):
                old = s["index"][:, 0, :, side].view(_E4M3).float() * _pow2(less)[..., None]
                old = old.to(_E4M3).float().masked_fill(anew[..., None], none)
                s["index"][:, 0, :, side] = old.scatter_reduce(0, to, new.float(), reduce).to(_E4M3).view(torch.uint8)
    return _append_outputs(s)


def _read_plain(s):
    page, off = s["slots"] // PAGE, s["slots"] % PAGE
    d = s["case"]["d"]
    k = s["k_pool"][:, 0].unflatten(-1, (PAGE, d))[page, :, off]
    v = s["v_pool"][:, 0].unflatten(-1, (4, d, 4))[page, :, off // 4, :, off % 4]
    for x, side, out in ((k, 0, s["k_out"]), (v, 1, s["v_out"])):
        out.copy_((x.view(_E4M3).float() * s["scales"][page, 0, :, side][..., None]).flatten(1))
    return s["k_out"], s["v_out"]


def _attn_plain(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, n, most = hq // hkv, case["batch"], s["max_rows"]
    rows = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu"][1:].contiguous(), rows.int(), right=True)
    i = rows - s["cu"][b]
    q = torch.zeros((n, most, hkv, g, d), device="cuda")
    q[b, i] = s["q"].float().view(-1, hkv, g, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, hkv, most * g, d)
    at = s["tables"][:, :-(-s["max_ctx"] // PAGE)].long()
    k = _values(s["k_pool"][at, 1], s["scales"][at, 1, :, 0], False).transpose(1, 2).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del k
    last = (s["start"][:, None] + torch.arange(most, device="cuda")).repeat_interleave(g, 1)
    hidden = torch.arange(score.shape[-1], device="cuda") > last[:, None, :, None]
    score.masked_fill_(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    v = _values(s["v_pool"][at, 1], s["scales"][at, 1, :, 1], True).transpose(1, 2).flatten(2, 3)
    o = torch.matmul(p, v).view(n, hkv, most, g, d).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o[b, i].flatten(1))
    return s["out"]


def _sparse_plain(s):
    case = s["case"]
    hq, hkv, d, n, budget = case["hq"], case["hkv"], case["d"], case["batch"], case["budget"]
    g = hq // hkv
    q = s["q"].float().view(n, hkv, g, d)
    at = s["tables"][:, :-(-s["max_ctx"] // PAGE)].long()
    # q in 8 bits, a power of two for every 32 dimensions; bounds in whole code units: every product's
    # sum is a whole number below 2^24, and only the groups' sums are rounded
    parts = q.unflatten(-1, (-1, 32))
    e = _exponent(parts.abs().amax(-1), 127.0)
    parts = (parts * _pow2(-e)[..., None]).round()
    bound = s["index"][at, 1].view(_E4M3).float().round().unflatten(-1, (-1, 32))  # [n, pages, hkv, 2, d / 32, 32]
    score = 0
    for j in range(d // 32):
        x = torch.cat([parts[..., j, :].clamp(min=0), parts[..., j, :].clamp(max=0)], -1)
        y = bound[..., j, :].flatten(-2).permute(0, 2, 3, 1).contiguous()
        score = score + torch.matmul(x, y) * _pow2(e[..., j])[..., None]
    score = score.amax(2) * s["scales"][at, 1, :, 0].transpose(1, 2)
    last = (s["start"] // PAGE)[:, None, None]
    p = torch.arange(at.shape[1], device="cuda")
    score = score.masked_fill((p < FIRST) | (p > last - RECENT), math.inf).masked_fill(p > last, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    chosen = torch.full((n, hkv, budget), 1 << 30, device="cuda")
    width = min(budget, at.shape[1])
    chosen[..., :width] = order[..., :width]
    chosen = chosen.masked_fill(chosen > last, 1 << 30).sort(-1).values
    none = chosen == 1 << 30
    s["pages"].copy_(chosen.masked_fill(none, -1))
    page = s["tables"][torch.arange(n, device="cuda")[:, None, None], chosen.masked_fill(none, 0)].long()
    h = torch.arange(hkv, device="cuda")[None, :, None]
    k = _values(s["k_pool"][page, 1, h], s["scales"][page, 1, h, 0], False).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    pos = (chosen[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(2)
    score = score.masked_fill((pos > s["start"][:, None, None])[:, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    v = _values(s["v_pool"][page, 1, h], s["scales"][page, 1, h, 1], True).flatten(2, 3)
    s["out"].copy_(torch.matmul(p, v).flatten(1))
    return s["pages"], s["out"]


# ---- the framework's calls ----------------------------------------------------------------

_LIB = {}


def _lib():
    """The library's handle on the current device, as a program keeps it."""
    if not _LIB:
        import __graft_entry__
        _LIB["lib"] = __graft_entry__.load_package().library.default(torch.cuda.current_device())
    return _LIB["lib"]


def _append_own(s):
    case, lib = s["case"], _lib()
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    qkv, bias = s["qkv"], s["bias"]
    a, b = hq * d, (hq + hkv) * d
    biases = {} if bias is None else {"q_bias": bias[:a], "k_bias": bias[a:b], "v_bias": bias[b:]}
    lib.kv8_append(qkv[:, :a], qkv[:, a:b], qkv[:, b:], s["cos"], s["sin"], s["positions"], s["slots"],
                   s["k_pool"], s["v_pool"], s["scales"], 0, 1, hq, hkv, d, bounds=s["index"],
                   q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"], **biases)
    return _append_outputs(s)


def _read_own(s):
    case = s["case"]
    _lib().kv8_read(s["k_out"], s["v_out"], s["slots"], s["k_pool"], s["v_pool"], s["scales"], 0, 1, case["hkv"],
                    case["d"])
    return s["k_out"], s["v_out"]


def _attn_own(s):
    case, lib = s["case"], _lib()
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["batch"]
    rows = s["q"].shape[0]
    if "workspace" not in s:  # one for every call of these sizes, as a program keeps it
        s["workspace"] = lib.kv8_workspace(n, rows, s["max_rows"], s["max_ctx"], hq, hkv, d)
    lib.kv8_attention(s["out"], s["q"], s["k_pool"], s["v_pool"], s["scales"], s["tables"], s["start"], n, rows,
                      s["max_rows"], s["max_ctx"], 1, 2, hq, hkv, d, 1.0 / math.sqrt(d),
                      cu_seqlens=s["cu"], workspace=s["workspace"])
    return s["out"]


def _sparse_own(s):
    case, lib = s["case"], _lib()
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["batch"]
    if "workspace" not in s:
        s["workspace"] = lib.kv8_sparse_workspace(n, s["max_ctx"], case["budget"], hq, hkv, d)
    lib.kv8_select(s["pages"], s["q"], s["index"], s["scales"], s["tables"], s["start"], n, s["max_ctx"], FIRST,
                   RECENT, 1, 2, hq, hkv, d, workspace=s["workspace"])
    lib.kv8_sparse_attention(s["out"], s["q"], s["k_pool"], s["v_pool"], s["scales"], s["tables"], s["start"],
                             s["pages"], n, s["max_ctx"], 1, 2, hq, hkv, d, 1.0 / math.sqrt(d),
                             workspace=s["workspace"])
    return s["pages"], s["out"]


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    hkv, d = case["hkv"], case["d"]
    if case["kind"] == "read":
        rows = case["rows"]
        return {"bytes": rows * (6.0 * hkv * d + 8) + -(-rows // PAGE) * 8.0 * hkv, "flops": 2.0 * rows * hkv * d}
    hq = case["hq"]
    if case["kind"] == "append":
        rows = case["rows"]
        decode = rows == case["seqs"]
        row = 2.0 * (2 * hq + 2 * hkv) * d + 12 + 2.0 * hkv * d
        # scales and key bounds: written, and read where a page goes on
        page = (2.0 * d + 8) * hkv * (2 if decode else 1)
        pages = rows if decode else rows / PAGE
        return {"bytes": rows * (row + d * 4.0) + pages * page, "flops": 8.0 * rows * (hq + hkv) * d}
    held, new = (x.astype(np.float64) for x in _lengths(case))
    rows = float(new.sum())
    if case["kind"] == "attn":
        keys = float((new * held + new * (new + 1) / 2).sum())
        pages = float(_pages(held + new).sum())
        return {"bytes": float((held + new).sum()) * hkv * 2 * d + pages * (8.0 * hkv + 4) + rows * 4 * hq * d,
                "flops": 4.0 * hq * d * keys}
    pages = _pages(held + 1).astype(np.float64)
    chosen = np.minimum(pages, case["budget"])
    return {"bytes": float(pages.sum()) * ((2.0 * d + 4) * hkv + 4) +
            float(chosen.sum()) * hkv * (PAGE * 2.0 * d + 8 + 4) + rows * 4 * hq * d,
            "flops": 4.0 * hq * d * float(pages.sum() + PAGE * chosen.sum())}


# ---- the same in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(_prepare_append(case, seed))
    if case["kind"] == "read":
        return _exact_read(_prepare_read(case, seed))
    return _exact_attn(_prepare_attn(case, seed))


def _exact_head(x, bias, norm, cos, sin):
    """One head's rows x [rows, d]: bias, norm, rotation."""
    x = x.double() if bias is None else x.double() + bias.double()
    if norm is not None:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    if cos is None:
        return x
    h = x.shape[-1] // 2
    return torch.cat([x[:, :h] * cos - x[:, h:] * sin, x[:, h:] * cos + x[:, :h] * sin], -1)


def _exact_code(x):
    """x [..] (at most 448 in size) to the nearest of e4m3's values, ties to the even one, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _code_values(slab):
    """The e4m3 values of bytes, from their bits, in 64 bits."""
    b = slab.long()
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m * 2.0 ** -9)
    return torch.where(b >= 128, -x, x)


def _exact_tokens(slab, is_v):
    """Code values [pages, 16, d] of one head's slabs [pages, 16 d]."""
    d = slab.shape[-1] // PAGE
    x = _code_values(slab)
    if not is_v:
        return x.view(-1, PAGE, d)
    out = torch.empty((slab.shape[0], PAGE, d), dtype=torch.float64, device=slab.device)
    for t in range(PAGE):
        out[:, t] = x[:, torch.arange(d, device=slab.device) * 4 + (t // 4) * 4 * d + t % 4]
    return out


def _exact_append(s):
    case, dt = s["case"], s["q_out"].dtype
    hq, hkv, d, rows = case["hq"], case["hkv"], case["d"], case["rows"]
    cos, sin = (t[s["positions"].long()].double() for t in (s["cos"], s["sin"]))
    slots = s["slots"].cpu().numpy()
    row_of = np.full((s["k_pool"].shape[0], PAGE), -1)  # the row that a token of a page comes from
    row_of[slots // PAGE, slots % PAGE] = np.arange(rows)
    row_of = torch.from_numpy(row_of).cuda()
    new = row_of >= 0
    here, anew = new.any(1), new[:, 0]
    q = []
    out = {"k": torch.empty(s["k_pool"].shape, dtype=torch.float64, device="cuda"),
           "v": torch.empty(s["v_pool"].shape, dtype=torch.float64, device="cuda"),
           "scales": s["scales"].double(), "bounds": torch.empty(s["index"].shape, dtype=torch.float64, device="cuda")}
    for h in range(hq + 2 * hkv):
        x = s["qkv"][:, h * d:(h + 1) * d]
        b = None if s["bias"] is None else s["bias"][h * d:(h + 1) * d]
        if h < hq:
            q.append(_exact_head(x, b, s["q_norm"], cos, sin))
            continue
        is_v, kv = (h - hq) // hkv, (h - hq) % hkv
        x = _exact_head(x, b, None, None, None) if is_v else _exact_head(x, b, s["k_norm"], cos, sin)
        x = x.to(dt).double().clamp(-LIMIT, LIMIT)
        x = torch.where(new[..., None], x[row_of.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))
        pool = s["v_pool" if is_v else "k_pool"][:, 0, kv]
        old = s["scales"][:, 0, kv, is_v].double()
        need = torch.exp2(torch.ceil(torch.log2((x.abs().amax((1, 2)) / 448).clamp(min=2.0 ** LEAST))))
        scale = torch.where(here, torch.where(anew, need, torch.maximum(need, old)), old)
        less = torch.where(anew, torch.ones_like(old), old / scale)[:, None, None]
        held = _exact_code(_exact_tokens(pool, is_v) * less)
        codes = torch.where(new[..., None], _exact_code(x / scale[:, None, None]), held)
        out["scales"][:, 0, kv, is_v] = scale
        if is_v:
            for t in range(PAGE):
                out["v"][:, 0, kv, torch.arange(d, device="cuda") * 4 + (t // 4) * 4 * d + t % 4] = codes[:, t]
            continue
        out["k"][:, 0, kv] = codes.flatten(1)
        for side, sign in ((0, 1.0), (1, -1.0)):
            most = (codes * sign).masked_fill(~new[..., None], -math.inf).amax(1)
            kept = _exact_code(_code_values(s["index"][:, 0, kv, side]) * less[:, 0]) * sign
            out["bounds"][:, 0, kv, side] = torch.where(anew[:, None], most, torch.maximum(most, kept)) * sign
    out["q"] = torch.cat(q, 1)
    return out


def _exact_read(s):
    case = s["case"]
    hkv, d = case["hkv"], case["d"]
    outs = []
    for pool, is_v in ((s["k_pool"], 0), (s["v_pool"], 1)):
        x = torch.empty((case["rows"], hkv, d), dtype=torch.float64, device="cuda")
        for h in range(hkv):
            v = _exact_tokens(pool[:, 0, h], is_v) * s["scales"][:, 0, h, is_v].double()[:, None, None]
            x[:, h] = v.view(-1, d)[s["slots"]]
        outs.append(x.flatten(1))
    return tuple(outs)


def _exact_attn(s):
    case = s["case"]
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["batch"]
    g = hq // hkv
    sparse = case["kind"] == "sparse"
    out = torch.empty((s["q"].shape[0], hq, d), dtype=torch.float64, device="cuda")
    cu, start = s["cu"].tolist(), s["start"].tolist()
    q = s["q"].double().view(-1, hq, d)
    for h in range(hkv):
        # every page of the pool once, then the sequences' own
        keys = _exact_tokens(s["k_pool"][:, 1, h], False) * s["scales"][:, 1, h, 0].double()[:, None, None]
        values = _exact_tokens(s["v_pool"][:, 1, h], True) * s["scales"][:, 1, h, 1].double()[:, None, None]
        for b in range(n):
            rows = cu[b + 1] - cu[b]
            ctx = start[b] + rows
            pages = s["tables"][b, :-(-ctx // PAGE)].long()
            at = torch.arange(len(pages), device="cuda")
            if sparse:
                at = _exact_choice(s, b, h, pages)
            k, v = keys[pages[at]].view(-1, d), values[pages[at]].view(-1, d)
            kt = k.t().contiguous()
            at = (at[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(1, -1)
            limit = (start[b] + torch.arange(rows, device="cuda"))[:, None]
            seen = at <= limit
            v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
            for j in range(h * g, (h + 1) * g):
                score = torch.matmul(q[cu[b]:cu[b + 1], j], kt) / math.sqrt(d)
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                out[cu[b]:cu[b + 1], j] = torch.matmul(torch.softmax(score, -1), v)
    if sparse:
        return None, out.flatten(1)  # (pages: whole numbers)
    return out.flatten(1)


def _exact_choice(s, b, h, pages):
    """The logical pages that sequence b's row reads with kv head h, ascending: by the definition of the
    score, whose sum over the groups of 32 dimensions is one in fp32."""
    case = s["case"]
    g, d = case["hq"] // case["hkv"], case["d"]
    bounds = torch.round(_code_values(s["index"][pages, 1, h]))  # [pages, 2, d]
    best = torch.full((len(pages),), -math.inf, device="cuda")
    for j in range(h * g, (h + 1) * g):
        x = s["q"][b, j * d:(j + 1) * d].double()
        score = torch.zeros(len(pages), device="cuda")
        for i in range(0, d, 32):
            y = x[i:i + 32]
            unit = torch.exp2(torch.ceil(torch.log2((y.abs().max() / 127).clamp(min=2.0 ** LEAST))))
            whole = torch.round(y / unit)
            top = torch.where(whole > 0, bounds[:, 0, i:i + 32], bounds[:, 1, i:i + 32])
            score = score + ((top * whole).sum(-1) * unit).float()
        best = torch.maximum(best, score)
    best = best * s["scales"][pages, 1, h, 0]
    best[:FIRST] = math.inf
    best[max(0, len(pages) - RECENT):] = math.inf
    rank = torch.argsort(-best, stable=True)[:case["budget"]]
    return rank.sort().values
