"""Host-side refusals of the page maps, the normed appends and the 4-bit attention, before any
GPU call (CPU only), sizes, and what their kernels keep in registers."""
import ctypes
import types

import pytest
import torch

from lucciola_rs_amd import library
from test_abi import kernel_metadata

P = ctypes.c_void_p


@pytest.fixture
def cdll():
    return library.load_cdll()


def call(fn, defaults, **kw):
    assert set(kw) <= set(defaults), kw
    rc = fn(*(defaults | kw).values())
    return rc


EXTEND = dict(ctx=P(1), stream=None, batch=4, new=P(64), lens=P(64), tables=P(64), stride=10, free=P(64),
              state=P(64), num_blocks=40, rows=8, slots=P(64), positions=P(64), cu=P(64), start=P(64))
TRUNCATE = dict(ctx=P(1), stream=None, batch=4, keep=P(64), lens=P(64), tables=P(64), stride=10, free=P(64),
                state=P(64), num_blocks=40)


def test_map_refusals(cdll):
    for fn, base, counts in ((cdll.luc_block_extend, EXTEND, "new"), (cdll.luc_block_truncate, TRUNCATE, "keep")):
        assert call(fn, base, ctx=None) == -1
        assert call(fn, base, batch=-1) == -1
        assert call(fn, base, batch=4097) == -2
        assert call(fn, base, stride=0) == -1
        assert call(fn, base, stride=(1 << 26) + 1) == -1
        assert call(fn, base, num_blocks=0) == -1
        for name in (counts, "lens", "tables", "free", "state"):
            assert call(fn, base, **{name: None}) == -1, name
        assert call(fn, base, batch=0) == 0
    f = cdll.luc_block_extend
    assert call(f, EXTEND, rows=-1) == -1
    for name in ("slots", "positions", "cu", "start"):
        assert call(f, EXTEND, **{name: None}) == -1, name
    assert call(f, EXTEND, slots=P(68)) == -1
    assert call(f, EXTEND, batch=0, rows=0, slots=None, positions=None) == 0


APPEND = dict(ctx=P(1), stream=None, dtype=0, q=P(64), k=P(64), v=P(64), stride=18 * 64, qb=None, kb=None, vb=None,
              qn=P(64), kn=P(64), eps=1e-6, cos=P(64), sin=P(64), max_pos=100, positions=P(64), slots=P(64), rows=3,
              q_out=P(64), q_out_stride=14 * 64, k_out=None, k_out_stride=0, k_pool=P(256), v_pool=P(256),
              num_blocks=8, layer=0, layers=2, hq=14, hkv=2, d=64, block=16)
APPEND4 = {}
for _k, _v in APPEND.items():
    if _k == "k_out_stride":
        APPEND4["v_out"] = None
    APPEND4[_k] = _v


@pytest.mark.parametrize("four", [False, True])
def test_append_refusals(cdll, four):
    fn, base = (cdll.luc_kv4_append, APPEND4) if four else (cdll.luc_qk_norm_rope_append, APPEND)
    c = lambda **kw: call(fn, base, **kw)  # noqa: E731
    assert c(ctx=None) == -1
    assert c(dtype=2) == -1
    assert c(d=96) == -2
    assert c(hq=15) == -1
    assert c(hq=18) == -2
    assert c(hkv=0) == -1
    assert c(block=32) == -2
    assert c(layer=2) == -1 and c(layer=-1) == -1 and c(layers=0) == -1
    assert c(num_blocks=0) == -1
    assert c(max_pos=0) == -1
    assert c(rows=-1) == -1
    for name in ("q", "k", "v", "q_out", "cos", "sin", "positions", "slots", "k_pool", "v_pool"):
        assert c(**{name: None}) == -1, name
    assert c(qn=None) == -1 and c(kn=None) == -1           # one without the other
    assert c(qn=None, kn=None, rows=0) == 0
    assert c(stride=14 * 64 - 8) == -1
    assert c(stride=18 * 64 + 4) == -1
    assert c(q_out_stride=14 * 64 - 8) == -1
    assert c(q_out_stride=14 * 64 + 4) == -1
    assert c(k_out=P(64), k_out_stride=64) == -1
    assert c(k_out=P(64), k_out_stride=132) == -1
    for name in ("q", "k", "v", "qb", "kb", "vb", "qn", "kn", "cos", "sin", "q_out", "k_out", "k_pool", "v_pool"):
        assert c(**{name: P(72), "k_out_stride": 128}) == -1, name
    assert c(slots=P(68)) == -1
    assert c(rows=0) == 0


ATTENTION = dict(ctx=P(1), stream=None, dtype=1, out=P(64), out_stride=14 * 64, q=P(64), q_stride=14 * 64,
                 k_pool=P(64), v_pool=P(64), tables=P(64), stride=32, num_blocks=100, cu=P(64), start=P(64), batch=3,
                 rows=9, max_rows=4, max_ctx=512, layer=1, layers=2, hq=14, hkv=2, d=64, block=16, scale=0.125,
                 ws=None, ws_bytes=0)


def test_attention_refusals(cdll):
    c = lambda **kw: call(cdll.luc_kv4_attention, ATTENTION, **kw)  # noqa: E731
    assert c(ctx=None) == -1
    assert c(dtype=-1) == -1
    assert c(d=256) == -2
    assert c(hq=13) == -1 and c(hq=18) == -2 and c(hkv=0) == -1
    assert c(block=8) == -2
    assert c(layer=2) == -1 and c(layers=0) == -1
    assert c(num_blocks=0) == -1
    assert c(batch=-1) == -1 and c(rows=-1) == -1 and c(max_rows=0) == -1
    assert c(max_ctx=0) == -1 and c(max_ctx=513) == -1 and c(max_ctx=(1 << 30) + 1, stride=1 << 27) == -1
    assert c(stride=0) == -1
    assert c(cu=None) == -1                                # 9 rows of 3 sequences
    for name in ("out", "q", "k_pool", "v_pool", "tables", "start"):
        assert c(**{name: None}) == -1, name
    assert c(q_stride=13 * 64) == -1 and c(q_stride=14 * 64 + 4) == -1
    assert c(out_stride=13 * 64) == -1 and c(out_stride=14 * 64 + 2) == -1
    assert c(q=P(72)) == -1 and c(out=P(68)) == -1 and c(k_pool=P(72)) == -1 and c(v_pool=P(72)) == -1
    assert c(rows=1 << 28) == -1                           # rows x heads past 2^31
    assert c(hq=1 << 21, hkv=1 << 20, q_stride=1 << 40, out_stride=1 << 40, rows=3, cu=None) == -1
    assert c(batch=0) == 0 and c(rows=0) == 0
    big = dict(stride=4096, max_ctx=65536)
    need = cdll.luc_kv4_workspace_size(3, 9, 4, 65536, 14, 2, 64)
    assert need > 0
    assert c(**big) == -5
    assert c(**big, ws=P(4096), ws_bytes=need - 4) == -5
    assert c(**big, ws=P(4096 + 64), ws_bytes=need) == -1


def test_sizes(cdll):
    assert cdll.luc_kv4_page_bytes(64) == 640 and cdll.luc_kv4_page_bytes(128) == 1280
    assert cdll.luc_kv4_page_bytes(96) == 0
    ws = cdll.luc_kv4_workspace_size
    assert ws(1, 1, 1, 16, 14, 2, 64) == 0                 # one split
    for bad in ((0, 1, 1, 16, 14, 2, 64), (1, 0, 1, 16, 14, 2, 64), (1, 1, 0, 16, 14, 2, 64), (1, 1, 1, 0, 14, 2, 64),
                (1, 1, 1, 9999, 15, 2, 64), (1, 1, 1, 9999, 18, 2, 64), (1, 1, 1, 9999, 14, 2, 96),
                (1, 1, 1, (1 << 30) + 1, 14, 2, 64), (1, 1 << 28, 1, 4096, 14, 2, 64), (9, 9, 1, 4096, 1 << 24, 1 << 24, 64),
                ((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1, 1 << 30, 8, 1, 64)):
        assert ws(*bad) == 0
    # the largest call's workspace: a few partials a CU, not one a page
    assert ws(64, 64, 1, 1 << 20, 28, 4, 128) < 1 << 28
    assert ws(1, 512, 512, 1 << 20, 12, 2, 128) < 1 << 29


def test_binding_refusals():
    """Shapes, types and strides that the binding checks before a call (tensors on the CPU)."""
    lib = object.__new__(library.LucAttn)
    lib.lib, lib.ctx, lib.device = library.load_cdll(), ctypes.c_void_p(), -1  # (what a CPU tensor's device is)
    stream = types.SimpleNamespace(cuda_stream=0)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    ext = dict(new_tokens=i32(2), lens=i32(2), tables=i32(2, 4), free_list=i32(8), state=i32(4), slots=i64(5),
               positions=i32(5), cu_seqlens=i32(3), start_pos=i32(2),
               stream=stream)
    for k, v in dict(new_tokens=i64(2), lens=i32(1), tables=i64(2, 4), state=i32(3), slots=i32(5), positions=i32(4),
                     cu_seqlens=i32(2), start_pos=i32(1), free_list=i32(16)[::2]).items():
        with pytest.raises(ValueError):
            lib.block_extend(**(ext | {k: v}))
    with pytest.raises(ValueError):
        lib.block_truncate(i32(1), i32(2), i32(2, 4), i32(8), i32(4), stream=stream)
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    qkv = half(3, 8 * 64)
    q, k, v = qkv[:, :256], qkv[:, 256:384], qkv[:, 384:]
    cos = torch.zeros(10, 32)
    pool4 = torch.zeros(2, 1, 2, 640, dtype=torch.uint8)
    base = dict(q=q, k=k, v=v, cos=cos, sin=cos, positions=i32(3), slots=i64(3), k_pool=pool4, v_pool=pool4, layer=0,
                num_layers=1, hq=4, hkv=2, head_dim=64, stream=stream)
    for kw in (dict(q=q[:, :128]), dict(k=half(3, 128)), dict(v=v[:2]), dict(q_out=half(2, 256)), dict(cos=cos[:, :16]),
               dict(positions=i32(2)), dict(slots=i32(3)), dict(k_pool=pool4[..., :600]), dict(k_pool=half(2, 1, 2, 640)),
               dict(q_norm=half(32), k_norm=half(32)), dict(q_bias=half(128)), dict(k_out=half(3, 64)),
               dict(k_out=half(3, 128), v_out=half(3, 136)[:, :128])):
        with pytest.raises((TypeError, ValueError)):
            lib.kv4_append(**(base | kw))
    for kw in (dict(k=k.bfloat16()), dict(q_out=torch.zeros(3, 256)), dict(v_bias=torch.zeros(128))):
        with pytest.raises((TypeError, ValueError)):
            lib.kv4_append(**(base | kw))
    with pytest.raises((TypeError, ValueError)):
        lib.qk_norm_rope_append(**(base | dict(k_pool=torch.zeros(2, 1, 2, 16, 64), v_pool=half(2, 1, 2, 16, 64))))
    with pytest.raises(library.LucError, match="null context"):  # what is right reaches the library
        lib.kv4_append(**base)
    # one row from tensors of its own, or with any stride
    one = dict(q=half(1, 256), k=half(1, 128), v=half(1, 131)[:, :128], positions=i32(1), slots=i64(1), k_out=half(1, 128),
               v_out=half(1, 140)[:, :128])
    with pytest.raises(library.LucError, match="null context"):
        lib.kv4_append(**(base | one))
    with pytest.raises(ValueError, match="stride differ"):
        lib.kv4_append(**(base | dict(k=half(3, 128))))
    att = dict(out=half(3, 256), q=q, k_pool=pool4, v_pool=pool4, tables=i32(3, 2), start_pos=i32(3), batch=3,
               total_rows=3, max_rows=1, max_ctx=32, layer=0, num_layers=1, hq=4, hkv=2, head_dim=64, sm_scale=0.125, stream=stream)
    for kw in (dict(out=half(2, 256)), dict(out=torch.zeros(3, 256)), dict(q=half(3, 128)), dict(tables=i32(2, 2)),
               dict(start_pos=i32(2)), dict(cu_seqlens=i32(3)), dict(v_pool=pool4[:, :, :1]), dict(total_rows=4)):
        with pytest.raises((TypeError, ValueError)):
            lib.kv4_attention(**(att | kw))
    with pytest.raises(library.LucError, match="null context"):
        lib.kv4_attention(**att)
    lib.device = 0  # tensors of another device than the library's
    for call in (lambda: lib.block_extend(**ext), lambda: lib.block_truncate(i32(2), i32(2), i32(2, 4), i32(8), i32(4), stream=stream),
                 lambda: lib.kv4_append(**base), lambda: lib.kv4_attention(**att)):
        with pytest.raises((TypeError, ValueError), match="library's device"):
            call()


def test_kernels_keep_their_values_in_registers():
    for obj in ("block_map", "norm_append", "kv4_attention"):
        kernels = kernel_metadata(obj)
        assert kernels
        for kernel, spilled, scratch in kernels:
            assert (spilled, scratch) == (0, 0), kernel


def test_engine_refusals():
    """DeviceBlocks and Kv4Cache say what they were given wrongly before any launch."""
    import torch
    from lucciola_rs_amd.engine import DeviceBlocks, Kv4Cache
    from lucciola_rs_amd.library import LucError

    calls = []

    class Lib:
        def block_extend(self, *a, **kw):
            calls.append(a)

    for sizes in ((0, 1, 1, 1), (4, 0, 1, 1), (4, 1, 0, 1), (4, 1, 1, 0)):
        with pytest.raises(ValueError, match="must be positive"):
            DeviceBlocks(*sizes, device="cpu", lib=Lib())
    blocks = DeviceBlocks(4, 2, 3, 10, device="cpu", lib=Lib())
    assert blocks.free_list.tolist() == [3, 2, 1, 0] and blocks.num_free == 4
    new = torch.zeros(2, dtype=torch.int32)
    for rows in (-1, 11):
        with pytest.raises(ValueError, match="outside"):
            blocks.extend(new, rows=rows)
    assert not calls
    blocks.extend(new, rows=0)
    blocks.extend(new)
    assert [a[5].numel() for a in calls] == [0, 10]
    blocks.check()
    for status, code, text in ((1, -6, "pages"), (2, -1, "table row"), (5, -1, "out of range"), (8, -1, "rows")):
        blocks.state[1] = status
        with pytest.raises(LucError, match=text) as e:
            blocks.check()
        assert e.value.code == code
        blocks.check()
    with pytest.raises(LucError, match="head dimension"):
        Kv4Cache(1, 4, 2, 96, 4, 1, 64, device="cpu", lib=Lib())
