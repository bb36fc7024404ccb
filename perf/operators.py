"""A serving step over a paged cache held in 4 bits, operator by operator: what is called, on what, and its plain form.

- "map": pages for the new rows of a batch, on the GPU: block tables, the slot and position of
  every new row, and the roll-back of the same rows (`LucAttn.block_extend`, `block_truncate`).
- "append16": RMS norms of q's and k's heads, their rotation and the write of k and v into a
  16-bit paged pool by slot (`LucAttn.qk_norm_rope_append`).
- "append4": the same into a 4-bit pool (`LucAttn.kv4_append`).
- "attn4": attention of a batch's new rows over a 4-bit pool (`LucAttn.kv4_attention`), one row
  a sequence (decode steps) or packed prompts.

`own` chooses between the framework's calls and plain torch in `run`.  Pools of 4 bits hold, for
each page of 16 tokens, layer and kv head, 10 * d bytes: 8 * d of values in pairs, then 2 * d of
scales.  A group is 32 consecutive values of one token's head: value = n * s + m, s and m in fp16.
K: values [16 tokens][d / 2 bytes], the even dimension in the low half of a byte; then (s, m) as
[16 tokens][d / 32 groups][2].  V: values [2 halves of the page][d / 4][8 tokens][2 bytes], four
dimensions of a token in two bytes; then [2 halves][d / 32 groups][s, m][8 tokens].
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
GROUP = 32
EPS = 1e-6
ROPE_BASE = 1e6
LIMIT = 60000.0  # values beyond it are stored as it
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the next token of a small batch: the latency of a captured loop's bookkeeping
        {"name": "map_decode_b8", "kind": "map", "batch": 8, "held_lo": 100, "held_hi": 4000,
         "new_lo": 1, "new_hi": 1},
        # a burst of new prompts, ragged, some after a cached prefix
        {"name": "map_prompts_b64", "kind": "map", "batch": 64, "held_lo": 0, "held_hi": 2000,
         "new_lo": 17, "new_hi": 4001},
        # the new rows of a serving batch (the benchmark's decode workload), 16-bit cache
        {"name": "append16_b32", "kind": "append16", "rows": 32, "seqs": 32, "hq": 14, "hkv": 2,
         "d": 64, "dtype": "f16", "norm": True, "bias": False},
        # four long prompts, 16-bit cache
        {"name": "append16_prompts", "kind": "append16", "rows": 8191, "seqs": 4, "hq": 28,
         "hkv": 4, "d": 128, "dtype": "bf16", "norm": True, "bias": False},
        # the new rows of a full serving batch, 4-bit cache, projections with biases
        {"name": "append4_b64", "kind": "append4", "rows": 64, "seqs": 64, "hq": 28, "hkv": 4,
         "d": 128, "dtype": "bf16", "norm": False, "bias": True},
        # ragged prompts, 4-bit cache
        {"name": "append4_prompts", "kind": "append4", "rows": 4100, "seqs": 5, "hq": 14,
         "hkv": 2, "d": 64, "dtype": "f16", "norm": True, "bias": False},
        # one sequence, short context: the latency of a chat's next token
        {"name": "attn4_single", "kind": "attn4", "batch": 1, "lo": 512, "hi": 512, "rows_lo": 1,
         "rows_hi": 1, "hq": 14, "hkv": 2, "d": 64, "dtype": "f16"},
        # a serving batch of mixed contexts (the benchmark's decode workload)
        {"name": "attn4_b32_mixed", "kind": "attn4", "batch": 32, "lo": 128, "hi": 4096,
         "rows_lo": 1, "rows_hi": 1, "hq": 14, "hkv": 2, "d": 64, "dtype": "f16"},
        # few sequences of long documents
        {"name": "attn4_b8_32k", "kind": "attn4", "batch": 8, "lo": 30000, "hi": 32768,
         "rows_lo": 1, "rows_hi": 1, "hq": 12, "hkv": 2, "d": 128, "dtype": "bf16"},
        # the largest decode: a full batch of long mixed contexts
        {"name": "attn4_b64_long", "kind": "attn4", "batch": 64, "lo": 1024, "hi": 16384,
         "rows_lo": 1, "rows_hi": 1, "hq": 28, "hkv": 4, "d": 128, "dtype": "bf16"},
        # a chunk of a long prompt after its cached prefix
        {"name": "attn4_chunk", "kind": "attn4", "batch": 1, "lo": 8000, "hi": 8000,
         "rows_lo": 512, "rows_hi": 512, "hq": 12, "hkv": 2, "d": 128, "dtype": "f16"},
        # long prompts of odd lengths from an empty cache
        {"name": "attn4_prompts", "kind": "attn4", "batch": 4, "lo": 0, "hi": 0, "rows_lo": 1531,
         "rows_hi": 2048, "hq": 14, "hkv": 2, "d": 64, "dtype": "bf16"},
    ]


# head layouts in use: (query heads, kv heads, head_dim)
_HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 8, 64), (32, 8, 128), (4, 2, 64),
          (8, 8, 128), (16, 2, 128)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["map"] * 2 + ["append16"] * 2 + ["append4"] * 2 + ["attn4"] * 6)
    if kind == "map":
        batch = _log_int(rng, 1, 256)
        new = rng.choice([1, _log_int(rng, 1, 120000 // batch)])
        held = rng.choice([0, _log_int(rng, 1, 8000)])
        return {"kind": kind, "batch": batch, "held_lo": held // 3, "held_hi": held,
                "new_lo": rng.choice([0, new]) if batch > 1 else new, "new_hi": new}
    hq, hkv, d = rng.choice(_HEADS)
    dtype = rng.choice(["f16", "bf16"])
    if kind in ("append16", "append4"):
        rows = _log_int(rng, 1, 8191 * 28 * 128 // (hq * d) if hq * d > 3584 else 8191)
        return {"kind": kind, "rows": rows, "seqs": min(rows, rng.choice([1, 3, 8, 64])),
                "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "norm": rng.choice([True, True, False]),
                "bias": rng.choice([True, False])}
    if rng.random() < 0.55:  # decode steps
        hi = _log_int(rng, 1, 32768)
        # at most 0.5 M tokens x heads x dimensions of 128
        batch = _log_int(rng, 1, max(1, min(64, 64 * 8700 * 4 * 128 // (hi * hkv * d))))
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
    if case["kind"] == "map":
        return (_spread(case["held_lo"], case["held_hi"], n, 0),
                _spread(case["new_lo"], case["new_hi"], n, 1000))
    rows = _spread(case["rows_lo"], case["rows_hi"], n, 1000)
    held = _spread(case["lo"], case["hi"], n, 0)
    if case["rows_hi"] == 1:
        held = held - 1  # lo .. hi are the contexts, the new row's own token among them
    return held, rows


def _int32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _pages(tokens):
    return -(-np.asarray(tokens, dtype=np.int64) // PAGE)


def _deal(seed, held, total):
    """Tables with the pages of `held` tokens dealt from a shuffled pool, room for `total`, and the
    rest of the pool (enough for `total`, and some): (tables, free list, pages in the pool)."""
    hp, tp = _pages(held), _pages(total)
    count = int(tp.sum() * 1.05) + 3
    perm = np.random.default_rng(int(seed)).permutation(count).astype(np.int32)
    tables = np.zeros((len(hp), max(1, int(tp.max()))), np.int32)
    starts = np.cumsum(hp) - hp
    for b in range(len(hp)):
        tables[b, :hp[b]] = perm[starts[b]:starts[b] + hp[b]]
    free = np.zeros(count, np.int32)
    free[:count - int(hp.sum())] = perm[int(hp.sum()):]
    return tables, free, count


def _rope_table(n, d):
    """cos and sin [n][d / 2] in fp32, as the engine keeps them."""
    i = np.arange(d // 2, dtype=np.float32) * np.float32(2) / np.float32(d)
    freq = np.power(np.float32(ROPE_BASE), i, dtype=np.float32)
    theta = (np.arange(n, dtype=np.float32)[:, None] / freq[None]).astype(np.float64)
    return (torch.from_numpy(np.cos(theta).astype(np.float32)).cuda(),
            torch.from_numpy(np.sin(theta).astype(np.float32)).cuda())


def prepare(case, seed):
    if case["kind"] == "map":
        return _prepare_map(case, seed)
    if case["kind"] == "attn4":
        return _prepare_attn(case, seed)
    return _prepare_append(case, seed)


def _prepare_map(case, seed):
    held, new = _lengths(case)
    tables, free, count = _deal(seed, held, held + new)
    n, rows = case["batch"], int(new.sum())
    state = torch.zeros(8, dtype=torch.int32, device="cuda")
    state[0] = count - int(_pages(held).sum())  # pages on the free list
    return {"case": case, "new": _int32(new), "keep": _int32(held), "lens": _int32(held),
            "tables": _int32(tables), "free": _int32(free), "state": state,
            "slots": torch.zeros(rows, dtype=torch.int64, device="cuda"),
            "positions": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "cu": torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
            "start": torch.zeros(n, dtype=torch.int32, device="cuda")}


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
    max_pos = int(pos.max()) + 1
    cos, sin = _rope_table(max_pos, d)
    qkv = _normal(gen, (rows, (hq + 2 * hkv) * d), 1.4, dt)
    s = {"case": case, "qkv": qkv, "cos": cos, "sin": sin, "positions": _int32(pos),
         "slots": torch.from_numpy(slots.astype(np.int64)).cuda(),
         "q_norm": _normal(gen, (d,), 0.1, dt, 1.0) if case["norm"] else None,
         "k_norm": _normal(gen, (d,), 0.1, dt, 1.0) if case["norm"] else None,
         "bias": _normal(gen, ((hq + 2 * hkv) * d,), 0.1, dt) if case["bias"] else None,
         "q_out": torch.zeros((rows, hq * d), dtype=dt, device="cuda")}
    if case["kind"] == "append16":
        shape, pool_dt = (len(pages), 1, hkv, PAGE, d), dt
    else:
        shape, pool_dt = (len(pages), 1, hkv, 10 * d), torch.uint8
        # the values that the cache holds for the new rows, as prompt attention reads them
        s["k_out"] = torch.zeros((rows, hkv * d), dtype=dt, device="cuda")
        s["v_out"] = torch.zeros((rows, hkv * d), dtype=dt, device="cuda")
    s["k_pool"] = torch.zeros(shape, dtype=pool_dt, device="cuda")
    s["v_pool"] = torch.zeros(shape, dtype=pool_dt, device="cuda")
    return s


# q and k of this size give scores of standard deviation about 2, as trained heads do
_QK_STD, _V_STD = 1.4, 1.0


def _pool4(gen, pages, layers, hkv, d, std, is_v):
    """A 4-bit pool as earlier appends filled it, in pieces."""
    pool = torch.empty((pages, layers, hkv, 10 * d), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (layers * hkv * PAGE * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = torch.randn((n, layers, hkv, PAGE, d), generator=gen, device="cuda").mul_(std)
        nib, s, m, _ = _encode(x)
        pool[i:i + n] = _pack_pages(nib, s, m, is_v)
    return pool


def _prepare_attn(case, seed):
    gen, dt = _gen(seed), _DT[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    held, new = _lengths(case)
    tables, _, count = _deal(seed, held + new, held + new)
    cu = np.concatenate([[0], np.cumsum(new)])
    rows = int(cu[-1])
    return {"case": case, "q": _normal(gen, (rows, hq * d), _QK_STD, dt),
            "k_pool": _pool4(gen, count, 2, hkv, d, _QK_STD, False),
            "v_pool": _pool4(gen, count, 2, hkv, d, _V_STD, True),
            "tables": _int32(tables), "cu": _int32(cu), "start": _int32(held),
            "max_ctx": int((held + new).max()), "max_rows": int(new.max()),
            "out": torch.zeros((rows, hq * d), dtype=dt, device="cuda")}


# ---- the 4-bit format in plain torch ------------------------------------------------------

def _encode(x):
    """x [..., d] (values of a 16-bit type, as fp32): (n, s, m, the values they stand for)."""
    g = x.unflatten(-1, (-1, GROUP)).clamp(-LIMIT, LIMIT)
    m = g.amin(-1).half()
    s = ((g.amax(-1) - m.float()) / 15.0).clamp(min=0.0).half()
    sf, mf = s.float()[..., None], m.float()[..., None]
    n = torch.where(sf > 0, ((g - mf) / sf).round().clamp(0, 15), torch.zeros_like(g))
    return n.flatten(-2).to(torch.uint8), s, m, (n * sf + mf).flatten(-2)


def _pack_k(n):
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _pack_pages(n, s, m, is_v):
    """Slabs [..., 10 d] of n [..., 16, d] and s, m [..., 16, d / 32]."""
    by = _pack_k(n)  # [..., 16, d / 2]
    sm = torch.stack([s, m], -1)  # [..., 16, d / 32, 2]
    if is_v:
        by = by.unflatten(-1, (-1, 2)).unflatten(-3, (2, 8)).transpose(-3, -2)
        sm = sm.unflatten(-3, (2, 8)).movedim(-3, -1)
    return torch.cat([by.flatten(n.dim() - 2),
                      sm.contiguous().view(torch.uint8).flatten(n.dim() - 2)], -1)


def _unpack_pages(slab, is_v):
    """Values [..., 16, d] in fp32 of slabs [..., 10 d]."""
    d = slab.shape[-1] // 10
    by, sm = slab[..., :8 * d], slab[..., 8 * d:].contiguous().view(torch.float16)
    if is_v:
        by = by.unflatten(-1, (2, d // 4, 8, 2)).transpose(-3, -2).flatten(-4, -3)
        sm = sm.unflatten(-1, (2, d // GROUP, 2, 8)).movedim(-1, -3).flatten(-4, -3)
    by = by.reshape(*slab.shape[:-1], PAGE, d // 2)
    sm = sm.reshape(*slab.shape[:-1], PAGE, d // GROUP, 2).float()
    n = torch.stack([by & 15, by >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (n * sm[..., 0, None] + sm[..., 1, None]).flatten(-2)


# ---- one pass -----------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "map":
        return _map_own(state) if own else _map_plain(state)
    if kind == "attn4":
        return _attn_own(state) if own else _attn_plain(state)
    return _append_own(state) if own else _append_plain(state)


def _map_outputs(s):
    return {k: s[k] for k in ("slots", "positions", "cu", "start", "tables", "free", "lens")} | {
        "count": s["state"][:1]}


def _map_plain(s):
    lens, new, tables, free, state = s["lens"], s["new"], s["tables"], s["free"], s["state"]
    held, total = (lens + PAGE - 1) // PAGE, (lens + new + PAGE - 1) // PAGE
    need = total - held
    before = need.cumsum(0) - need
    s["cu"][1:] = new.cumsum(0)
    s["start"].copy_(lens)
    rows = torch.arange(s["slots"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu"][1:].contiguous(), rows.int(), right=True)
    pos = lens[b] + rows - s["cu"][b]
    page = pos // PAGE
    taken = free[(state[0] - 1 - (before[b] + page - held[b])).clamp(0, free.shape[0] - 1)]
    id_ = torch.where(page >= held[b], taken, tables[b, page])
    tables[b, page] = id_
    s["slots"].copy_(id_.long() * PAGE + pos % PAGE)
    s["positions"].copy_(pos)
    lens += new
    state[0] -= need.sum()
    out = {k: v.clone() for k, v in _map_outputs(s).items()}
    # the roll-back: the pages go back to the places that they came from
    keep = torch.minimum(s["keep"], lens)
    held, left = (lens + PAGE - 1) // PAGE, (keep + PAGE - 1) // PAGE
    gone = held - left
    after = gone.flip(0).cumsum(0).flip(0) - gone
    j = torch.arange(tables.shape[1], device="cuda")[None]
    back = (j >= left[:, None]) & (j < held[:, None])
    to = state[0] + after[:, None] + held[:, None] - 1 - j
    at = torch.where(back, to, torch.full_like(to, free.shape[0]))
    grown = torch.cat([free, free[:1]])
    grown[at.flatten()] = tables.flatten()
    free.copy_(grown[:-1])
    tables[back] = 0
    lens.copy_(keep)
    state[0] += gone.sum()
    return out, _map_outputs(s)


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
    k = torch.cat([k1 * c - k2 * n, k1 * n + k2 * c], -1).to(dt)
    v = v.to(dt)
    page, off = s["slots"] // PAGE, s["slots"] % PAGE
    if case["kind"] == "append16":
        s["k_pool"][page, 0, :, off] = k
        s["v_pool"][page, 0, :, off] = v
        return s["q_out"], s["k_pool"], s["v_pool"]
    kn, ks, km, kv = _encode(k.float())
    vn, vs, vm, vv = _encode(v.float())
    pool = s["k_pool"][:, 0]
    pool[..., :8 * d].unflatten(-1, (PAGE, d // 2))[page, :, off] = _pack_k(kn)
    pool[..., 8 * d:].view(torch.float16).unflatten(-1, (PAGE, d // GROUP, 2))[page, :, off] = \
        torch.stack([ks, km], -1)
    pool = s["v_pool"][:, 0]
    pool[..., :8 * d].unflatten(-1, (2, d // 4, 8, 2))[page, :, off // 8, :, off % 8] = \
        _pack_k(vn).unflatten(-1, (-1, 2))
    pool[..., 8 * d:].view(torch.float16).unflatten(-1, (2, d // GROUP, 2, 8))[
        page, :, off // 8, :, :, off % 8] = torch.stack([vs, vm], -1)
    s["k_out"].copy_(kv.flatten(1))
    s["v_out"].copy_(vv.flatten(1))
    return s["q_out"], s["k_out"], s["v_out"]


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
    k = _unpack_pages(s["k_pool"][at, 1], False).transpose(1, 2).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del k
    last = (s["start"][:, None] + torch.arange(most, device="cuda")).repeat_interleave(g, 1)
    hidden = torch.arange(score.shape[-1], device="cuda") > last[:, None, :, None]
    score.masked_fill_(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    v = _unpack_pages(s["v_pool"][at, 1], True).transpose(1, 2).flatten(2, 3)
    o = torch.matmul(p, v).view(n, hkv, most, g, d).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o[b, i].flatten(1))
    return s["out"]


# ---- the framework's calls ----------------------------------------------------------------

_LIB = {}


def _lib():
    """The library's handle on the current device, as a program keeps it."""
    if not _LIB:
        import __graft_entry__
        _LIB["lib"] = __graft_entry__.load_package().library.default(torch.cuda.current_device())
    return _LIB["lib"]


def _map_own(s):
    lib = _lib()
    lib.block_extend(s["new"], s["lens"], s["tables"], s["free"], s["state"], s["slots"],
                     s["positions"], s["cu"], s["start"])
    out = {k: v.clone() for k, v in _map_outputs(s).items()}
    lib.block_truncate(s["keep"], s["lens"], s["tables"], s["free"], s["state"])
    return out, _map_outputs(s)


def _append_own(s):
    case, lib = s["case"], _lib()
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    qkv, bias = s["qkv"], s["bias"]
    a, b = hq * d, (hq + hkv) * d
    biases = {} if bias is None else {"q_bias": bias[:a], "k_bias": bias[a:b], "v_bias": bias[b:]}
    if case["kind"] == "append16":
        lib.qk_norm_rope_append(qkv[:, :a], qkv[:, a:b], qkv[:, b:], s["cos"], s["sin"],
                                s["positions"], s["slots"], s["k_pool"], s["v_pool"], 0, 1, hq, hkv,
                                d, q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                q_out=s["q_out"], **biases)
        return s["q_out"], s["k_pool"], s["v_pool"]
    lib.kv4_append(qkv[:, :a], qkv[:, a:b], qkv[:, b:], s["cos"], s["sin"], s["positions"],
                   s["slots"], s["k_pool"], s["v_pool"], 0, 1, hq, hkv, d, q_norm=s["q_norm"],
                   k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"], k_out=s["k_out"],
                   v_out=s["v_out"], **biases)
    return s["q_out"], s["k_out"], s["v_out"]


def _attn_own(s):
    case, lib = s["case"], _lib()
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["batch"]
    rows = s["q"].shape[0]
    if "workspace" not in s:  # one for every call of these sizes, as a program keeps it
        s["workspace"] = lib.kv4_workspace(n, rows, s["max_rows"], s["max_ctx"], hq, hkv, d)
    lib.kv4_attention(s["out"], s["q"], s["k_pool"], s["v_pool"], s["tables"], s["start"], n, rows,
                      s["max_rows"], s["max_ctx"], 1, 2, hq, hkv, d, 1.0 / math.sqrt(d),
                      cu_seqlens=s["cu"], workspace=s["workspace"])
    return s["out"]


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    if case["kind"] == "map":
        held, new = _lengths(case)
        n, rows = case["batch"], int(new.sum())
        pages = int((_pages(held + new) - _pages(held)).sum())
        # lengths and counts; a slot and a position a row; a page's id out, and back again
        return {"bytes": 4.0 * (8 * n + 1) + 12.0 * rows + 20.0 * pages, "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "attn4":
        held, new = (x.astype(np.float64) for x in _lengths(case))
        keys = float((new * held + new * (new + 1) / 2).sum())
        tokens = float((held + new).sum())
        return {"bytes": tokens * (hkv * 1.25 * d + 0.25) + float(new.sum()) * 4 * hq * d,
                "flops": 4.0 * hq * d * keys}
    rows = case["rows"]
    table = min(rows, 8191) * d * 4.0  # cos and sin rows
    row = 2.0 * (2 * hq + 2 * hkv) * d + 12
    if case["kind"] == "append16":
        row += 4.0 * hkv * d
    else:
        row += 1.25 * hkv * d + 4.0 * hkv * d  # the cache, and the values that it holds
    return {"bytes": rows * row + table, "flops": 8.0 * rows * (hq + hkv) * d}


# ---- the same in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "map":
        return None  # whole numbers
    if case["kind"] == "attn4":
        return _exact_attn(_prepare_attn(case, seed))
    return _exact_append(_prepare_append(case, seed))


def _exact_head(x, bias, norm, cos, sin):
    """One head's rows x [rows, d]: bias, norm, rotation."""
    x = x.double() if bias is None else x.double() + bias.double()
    if norm is not None:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    if cos is None:
        return x
    h = x.shape[-1] // 2
    return torch.cat([x[:, :h] * cos - x[:, h:] * sin, x[:, h:] * cos + x[:, :h] * sin], -1)


def _exact_stored(x):
    """What the cache holds of x [rows, d] (its 16-bit values, in 64 bits)."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[1], GROUP):
        y = x[:, g:g + GROUP].clamp(-LIMIT, LIMIT)
        m = y.min(1, keepdim=True).values.to(torch.float16).double()
        s = ((y.max(1, keepdim=True).values - m) / 15).clamp(min=0).to(torch.float16).double()
        n = torch.where(s > 0, torch.round((y - m) / s).clamp(0, 15), torch.zeros_like(y))
        out[:, g:g + GROUP] = n * s + m
    return out


def _exact_append(s):
    case, dt = s["case"], s["q_out"].dtype
    hq, hkv, d, rows = case["hq"], case["hkv"], case["d"], case["rows"]
    cos, sin = (t[s["positions"].long()].double() for t in (s["cos"], s["sin"]))
    q, k, v = [], [], []
    for h in range(hq + 2 * hkv):
        x = s["qkv"][:, h * d:(h + 1) * d]
        b = None if s["bias"] is None else s["bias"][h * d:(h + 1) * d]
        if h < hq:
            q.append(_exact_head(x, b, s["q_norm"], cos, sin))
        elif h < hq + hkv:
            k.append(_exact_head(x, b, s["k_norm"], cos, sin))
        else:
            v.append(_exact_head(x, b, None, None, None))
    q = torch.cat(q, 1)
    if case["kind"] == "append4":
        return (q, torch.cat([_exact_stored(x.to(dt).double()) for x in k], 1),
                torch.cat([_exact_stored(x.to(dt).double()) for x in v], 1))
    pools = []
    for x, pool in ((k, s["k_pool"]), (v, s["v_pool"])):
        p = pool.double()
        for h in range(hkv):
            p[s["slots"] // PAGE, 0, h, s["slots"] % PAGE] = x[h]
        pools.append(p)
    return q, pools[0], pools[1]


def _exact_values(slabs, d, is_v):
    """Tokens [pages * 16, d] in 64 bits of one head's slabs [pages, 10 d]."""
    sm = slabs[:, 8 * d:].contiguous().view(torch.float16).double()
    out = torch.empty((slabs.shape[0], PAGE, d), dtype=torch.float64, device=slabs.device)
    for t in range(PAGE):
        for x in range(d):
            g = x // GROUP
            if is_v:
                byte = ((t // 8) * (d // 4) + x // 4) * 16 + (t % 8) * 2 + (x % 4) // 2
                s_at = ((t // 8) * (d // GROUP) + g) * 16 + t % 8
                m_at = s_at + 8
            else:
                byte = t * (d // 2) + x // 2
                s_at = (t * (d // GROUP) + g) * 2
                m_at = s_at + 1
            n = (slabs[:, byte] >> 4 if x % 2 else slabs[:, byte] % 16).double()
            out[:, t, x] = n * sm[:, s_at] + sm[:, m_at]
    return out.view(-1, d)


def _exact_attn(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g = hq // hkv
    out = torch.empty((s["q"].shape[0], hq, d), dtype=torch.float64, device="cuda")
    cu, start = s["cu"].tolist(), s["start"].tolist()
    q = s["q"].double().view(-1, hq, d)
    for h in range(hkv):
        # every page of the pool once, then the sequences' own
        keys = _exact_values(s["k_pool"][:, 1, h], d, False).view(-1, PAGE, d)
        values = _exact_values(s["v_pool"][:, 1, h], d, True).view(-1, PAGE, d)
        for b in range(case["batch"]):
            n = cu[b + 1] - cu[b]
            ctx = start[b] + n
            pages = s["tables"][b, :-(-ctx // PAGE)].long()
            k, v = keys[pages].view(-1, d)[:ctx], values[pages].view(-1, d)[:ctx]
            kt = k.t().contiguous()
            at = torch.arange(ctx, device="cuda")[None]
            limit = (start[b] + torch.arange(n, device="cuda"))[:, None]
            for j in range(h * g, (h + 1) * g):
                score = torch.matmul(q[cu[b]:cu[b + 1], j], kt) / math.sqrt(d)
                score = torch.where(at <= limit, score, torch.full_like(score, -math.inf))
                out[cu[b]:cu[b + 1], j] = torch.matmul(torch.softmax(score, -1), v)
    return out.flatten(1)
