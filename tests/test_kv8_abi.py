"""Host-side refusals of the 8-bit cache's calls before any GPU call (CPU only), their sizes, what
their kernels keep in registers, and the plain forms that the GPU tests hold them to."""
import ctypes
import types

import numpy as np
import pytest
import torch

import kv8_ref as ref
from lucciola_rs_amd import library
from test_abi import kernel_metadata

P = ctypes.c_void_p


@pytest.fixture
def cdll():
    return library.load_cdll()


def call(fn, defaults, **kw):
    assert set(kw) <= set(defaults), kw
    return fn(*(defaults | kw).values())


APPEND = dict(ctx=P(1), stream=None, dtype=0, q=P(64), k=P(64), v=P(64), stride=18 * 64, qb=None, kb=None, vb=None,
              qn=P(64), kn=P(64), eps=1e-6, cos=P(64), sin=P(64), max_pos=100, positions=P(64), slots=P(64), rows=3,
              q_out=P(64), q_out_stride=14 * 64, k_pool=P(256), v_pool=P(256), scales=P(64), bounds=P(64),
              num_blocks=8, layer=0, layers=2, hq=14, hkv=2, d=64, block=16)
READ = dict(ctx=P(1), stream=None, dtype=1, k_out=P(64), v_out=P(64), stride=128, slots=P(64), rows=3, k_pool=P(64),
            v_pool=P(64), scales=P(64), num_blocks=8, layer=0, layers=2, hkv=2, d=64, block=16)
ATTENTION = dict(ctx=P(1), stream=None, dtype=1, out=P(64), out_stride=14 * 64, q=P(64), q_stride=14 * 64,
                 k_pool=P(64), v_pool=P(64), scales=P(64), tables=P(64), stride=32, num_blocks=100, cu=P(64),
                 start=P(64), batch=3, rows=9, max_rows=4, max_ctx=512, layer=1, layers=2, hq=14, hkv=2, d=64, block=16,
                 scale=0.125, ws=None, ws_bytes=0)
SELECT = dict(ctx=P(1), stream=None, dtype=1, pages=P(64), budget=40, first=1, recent=2, q=P(64), q_stride=14 * 64,
              bounds=P(64), scales=P(64), tables=P(64), stride=32, num_blocks=100, cu=P(64), start=P(64), batch=3,
              rows=3, max_ctx=512, layer=1, layers=2, hq=14, hkv=2, d=64, block=16, ws=None, ws_bytes=0)
SPARSE = dict(ctx=P(1), stream=None, dtype=1, out=P(64), out_stride=14 * 64, q=P(64), q_stride=14 * 64,
              k_pool=P(64), v_pool=P(64), scales=P(64), tables=P(64), stride=32, num_blocks=100, pages=P(64), budget=8,
              cu=P(64), start=P(64), batch=3, rows=3, max_ctx=512, layer=1, layers=2, hq=14, hkv=2, d=64, block=16,
              scale=0.125, ws=None, ws_bytes=0)


def sizes(c, group=True):
    assert c(ctx=None) == -1
    assert c(dtype=2) == -1 and c(dtype=-1) == -1
    assert c(d=96) == -2
    assert c(hkv=0) == -1
    assert c(block=32) == -2
    assert c(layer=2) == -1 and c(layer=-1) == -1 and c(layers=0) == -1
    assert c(num_blocks=0) == -1
    if group:
        assert c(hq=15) == -1 and c(hq=18) == -2


def test_append_refusals(cdll):
    c = lambda **kw: call(cdll.luc_kv8_append, APPEND, **kw)  # noqa: E731
    sizes(c)
    assert c(max_pos=0) == -1 and c(rows=-1) == -1
    for name in ("q", "k", "v", "q_out", "cos", "sin", "positions", "slots", "k_pool", "v_pool", "scales"):
        assert c(**{name: None}) == -1, name
    assert c(qn=None) == -1 and c(kn=None) == -1           # one without the other
    assert c(stride=14 * 64 - 8) == -1 and c(stride=18 * 64 + 4) == -1
    assert c(q_out_stride=14 * 64 - 8) == -1 and c(q_out_stride=14 * 64 + 4) == -1
    for name in ("q", "k", "v", "qb", "kb", "vb", "qn", "kn", "cos", "sin", "q_out", "k_pool", "v_pool", "bounds"):
        assert c(**{name: P(72)}) == -1, name
    assert c(slots=P(68)) == -1 and c(scales=P(68)) == -1 and c(positions=P(66)) == -1
    assert c(rows=1 << 27) == -1                           # threads past 2^32
    assert c(layers=1 << 21) == -1                         # a page past 2^32 bytes
    assert c(rows=0) == 0 and c(rows=0, q=None, k=None, v=None, q_out=None, positions=None, slots=None, bounds=None) == 0


def test_read_refusals(cdll):
    c = lambda **kw: call(cdll.luc_kv8_read, READ, **kw)  # noqa: E731
    sizes(c, group=False)
    assert c(rows=-1) == -1
    for name in ("k_out", "v_out", "slots", "k_pool", "v_pool", "scales"):
        assert c(**{name: None}) == -1, name
    assert c(stride=120) == -1 and c(stride=132) == -1
    for name in ("k_out", "v_out", "k_pool", "v_pool"):
        assert c(**{name: P(72)}) == -1, name
    assert c(slots=P(68)) == -1 and c(scales=P(68)) == -1
    assert c(rows=1 << 27) == -1
    assert c(rows=0) == 0 and c(rows=0, k_out=None, v_out=None, slots=None) == 0


def rows_of(c):
    assert c(batch=-1) == -1 and c(rows=-1) == -1
    assert c(max_ctx=0) == -1 and c(max_ctx=513) == -1 and c(max_ctx=(1 << 30) + 1, stride=1 << 27) == -1
    assert c(stride=0) == -1
    for name in ("q", "tables", "start", "scales"):
        assert c(**{name: None}) == -1, name
    assert c(q_stride=13 * 64) == -1 and c(q_stride=14 * 64 + 4) == -1
    assert c(q=P(72)) == -1 and c(scales=P(68)) == -1
    assert c(rows=1 << 28) == -1                           # rows x heads past 2^31
    assert c(layers=1 << 21) == -1
    assert c(batch=0) == 0


def test_attention_refusals(cdll):
    c = lambda **kw: call(cdll.luc_kv8_attention, ATTENTION, **kw)  # noqa: E731
    sizes(c)
    rows_of(c)
    assert c(max_rows=0) == -1
    assert c(cu=None) == -1                                # 9 rows of 3 sequences
    for name in ("out", "k_pool", "v_pool"):
        assert c(**{name: None}) == -1, name
    assert c(out_stride=13 * 64) == -1 and c(out_stride=14 * 64 + 2) == -1
    assert c(out=P(68)) == -1 and c(k_pool=P(72)) == -1 and c(v_pool=P(72)) == -1
    assert c(rows=0) == 0
    big = dict(stride=4096, max_ctx=65536)
    need = cdll.luc_kv8_workspace_size(3, 9, 4, 65536, 14, 2, 64)
    assert need > 0
    assert c(**big) == -5
    assert c(**big, ws=P(4096), ws_bytes=need - 4) == -5
    assert c(**big, ws=P(4096 + 64), ws_bytes=need) == -1


@pytest.mark.parametrize("sparse", [False, True])
def test_select_and_sparse_refusals(cdll, sparse):
    fn, base = (cdll.luc_kv8_sparse_attention, SPARSE) if sparse else (cdll.luc_kv8_select, SELECT)
    c = lambda **kw: call(fn, base, **kw)  # noqa: E731
    sizes(c)
    rows_of(c)
    assert c(cu=None, rows=4) == -1
    assert c(budget=0) == -1 and c(pages=None) == -1 and c(pages=P(66)) == -1
    assert c(batch=1 << 16, rows=1 << 16) == -2            # arrivals
    if sparse:
        for name in ("out", "k_pool", "v_pool"):
            assert c(**{name: None}) == -1, name
        assert c(out_stride=13 * 64) == -1 and c(out=P(68)) == -1
        assert c(rows=0) == 0
        big = dict(stride=4096, max_ctx=65536, budget=1000)
    else:
        assert c(first=-1) == -1 and c(recent=0) == -1 and c(first=39) == -1
        assert c(bounds=None) == -1 and c(bounds=P(72)) == -1
        big = dict(stride=4096, max_ctx=65536, budget=64)
    need = cdll.luc_kv8_sparse_workspace_size(3, 65536, big["budget"], 14, 2, 64)
    assert need > 0
    assert c(**big) == -5
    assert c(**big, ws=P(4096), ws_bytes=1 << 18) == -5
    assert c(**big, ws=P(4096 + 64), ws_bytes=need) == -1


def test_sizes(cdll):
    ws, sparse = cdll.luc_kv8_workspace_size, cdll.luc_kv8_sparse_workspace_size
    assert ws(1, 1, 1, 16, 14, 2, 64) == 0                 # one split
    for bad in ((0, 1, 1, 16, 14, 2, 64), (1, 0, 1, 16, 14, 2, 64), (1, 1, 0, 16, 14, 2, 64), (1, 1, 1, 0, 14, 2, 64),
                (1, 1, 1, 9999, 15, 2, 64), (1, 1, 1, 9999, 18, 2, 64), (1, 1, 1, 9999, 14, 2, 96),
                (1, 1, 1, (1 << 30) + 1, 14, 2, 64), (1, 1 << 28, 1, 4096, 14, 2, 64), (9, 9, 1, 4096, 1 << 24, 1 << 24, 64),
                ((1 << 31) - 1, (1 << 31) - 1, (1 << 31) - 1, 1 << 30, 8, 1, 64)):
        assert ws(*bad) == 0
    for bad in ((0, 9999, 8, 14, 2, 64), (1, 0, 8, 14, 2, 64), (1, 9999, 0, 14, 2, 64), (1, 9999, 8, 15, 2, 64),
                (1, 9999, 8, 14, 2, 32), (1, (1 << 30) + 1, 8, 14, 2, 64)):
        assert sparse(*bad) == 0
    assert sparse(4, 100, 7, 14, 2, 64) == 0               # no more pages than the budget, one split
    assert sparse(4, 113, 7, 14, 2, 64) == (1 << 18) + 4 * 2 * 8 * 4
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
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    qkv = half(3, 8 * 64)
    q, k, v = qkv[:, :256], qkv[:, 256:384], qkv[:, 384:]
    cos, pool, scales, bounds = torch.zeros(10, 32), u8(2, 1, 2, 1024), torch.zeros(2, 1, 2, 2), u8(2, 1, 2, 2, 64)
    app = dict(q=q, k=k, v=v, cos=cos, sin=cos, positions=i32(3), slots=i64(3), k_pool=pool, v_pool=pool, scales=scales,
               layer=0, num_layers=1, hq=4, hkv=2, head_dim=64, bounds=bounds, stream=stream)
    read = dict(k_out=half(3, 128), v_out=half(3, 128), slots=i64(3), k_pool=pool, v_pool=pool, scales=scales, layer=0,
                num_layers=1, hkv=2, head_dim=64, stream=stream)
    rows = dict(tables=i32(3, 2), start_pos=i32(3), batch=3, max_ctx=32, layer=0, num_layers=1, hq=4, hkv=2, head_dim=64,
                stream=stream)
    att = dict(out=half(3, 256), q=q, k_pool=pool, v_pool=pool, scales=scales, total_rows=3, max_rows=1, sm_scale=0.125) | rows
    sel = dict(pages=i32(3, 2, 4), q=q, bounds=bounds, scales=scales, first=1, recent=1) | rows
    spa = dict(out=half(3, 256), q=q, k_pool=pool, v_pool=pool, scales=scales, pages=i32(3, 2, 4), sm_scale=0.125) | rows
    pools = [dict(k_pool=pool[..., :1000]), dict(v_pool=pool[:1]), dict(k_pool=half(2, 1, 2, 1024)), dict(scales=scales[:1]),
             dict(scales=scales[..., :1]), dict(scales=scales.double()), dict(num_blocks=3)]
    for fn, base, bad in (
            (lib.kv8_append, app, pools + [
                dict(q=q[:, :128]), dict(k=half(3, 128)), dict(v=v[:2]), dict(q_out=half(2, 256)), dict(cos=cos[:, :16]),
                dict(positions=i32(2)), dict(slots=i32(3)), dict(q_norm=half(32), k_norm=half(32)), dict(q_bias=half(128)),
                dict(k=k.bfloat16()), dict(bounds=bounds[:1]), dict(bounds=half(2, 1, 2, 2, 64)), dict(bounds=u8(2, 1, 2, 128))]),
            (lib.kv8_read, read, pools + [
                dict(k_out=half(3, 120)), dict(v_out=half(2, 128)), dict(v_out=half(3, 136)[:, :128]), dict(slots=i64(2)),
                dict(slots=i32(3)), dict(v_out=torch.zeros(3, 128))]),
            (lib.kv8_attention, att, pools + [
                dict(out=half(2, 256)), dict(out=torch.zeros(3, 256)), dict(q=half(3, 128)), dict(tables=i32(2, 2)),
                dict(start_pos=i32(2)), dict(cu_seqlens=i32(3)), dict(total_rows=4)]),
            (lib.kv8_select, sel, [
                dict(pages=i32(3, 8)), dict(pages=i32(2, 2, 4)), dict(pages=i64(3, 2, 4)), dict(q=half(2, 256)), dict(q=half(3, 128)),
                dict(bounds=bounds[:1]), dict(scales=scales[..., :1]), dict(tables=i32(2, 2)), dict(start_pos=i32(2)),
                dict(cu_seqlens=i32(3)), dict(num_blocks=3)]),
            (lib.kv8_sparse_attention, spa, pools + [
                dict(pages=i32(3, 8)), dict(pages=i32(3, 1, 4)), dict(out=half(2, 256)), dict(q=half(2, 256)), dict(tables=i32(2, 2)),
                dict(start_pos=i32(2)), dict(cu_seqlens=i32(3))])):
        for kw in bad:
            with pytest.raises((TypeError, ValueError)):
                fn(**(base | kw))
        with pytest.raises(library.LucError, match="null context"):  # what is right reaches the library
            fn(**base)
        lib.device = 0  # tensors of another device than the library's
        with pytest.raises((TypeError, ValueError), match="library's device"):
            fn(**base)
        lib.device = -1


def test_kernels_keep_their_values_in_registers():
    for obj in ("kv8_append", "kv8_attention", "kv8_select"):
        kernels = kernel_metadata(obj)
        assert kernels
        for kernel, spilled, scratch in kernels:
            assert (spilled, scratch) == (0, 0), kernel


def test_engine_refusals():
    from lucciola_rs_amd.engine import Kv8Cache
    from lucciola_rs_amd.library import LucError
    with pytest.raises(LucError, match="head dimension"):
        Kv8Cache(1, 4, 2, 96, 4, 1, 64, device="cpu", lib=object())
    cache = Kv8Cache(1, 4, 2, 64, 4, 1, 64, device="cpu", lib=object())
    q = torch.zeros(1, 256)
    with pytest.raises(ValueError, match="bounds=True"):
        cache.attend_sparse(0, q, q, 64, 8)
    with pytest.raises(ValueError, match="rows to append"):
        cache.append(0, torch.zeros(2, 256), None, None, None)


def test_plain_forms():
    """The reference's own arithmetic: codes, exponents, slabs and choices by other means."""
    x = np.concatenate([np.linspace(-448, 448, 20001), 2.0 ** np.arange(-12, 9), -(2.0 ** -10) * np.arange(40)])
    x = x.astype(np.float32)
    cast = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert ref.equal_codes(ref.encode(x.astype(np.float64)), cast)
    assert np.array_equal(np.isnan(ref.TABLE), np.isin(np.arange(256), (127, 255)))
    assert ref.TABLE[126] == 448 and ref.TABLE[1] == 2.0 ** -9 and ref.TABLE[8] == 2.0 ** -6
    for a in (0.0, 1e-30, 447.0, 448.0, 448.5, 60000.0, 3.5, 3.5001, 1.75 * 2.0 ** -70):
        e = ref.exponent(a)
        assert e == ref.LEAST or a > 448 * 2.0 ** (e - 1)
        assert a <= 448 * 2.0 ** e and int(ref.exponents(np.array(a))) == e
    codes = np.arange(16 * 64, dtype=np.int64).reshape(16, 64).astype(np.uint8)
    assert np.array_equal(ref.of_slab(ref.v_slab(codes), True), codes)
    assert ref.v_slab(codes)[:4].tolist() == [int(codes[t, 0]) for t in range(4)]
    assert ref.choose(np.array([5, 1, 3, 3, 0, 2, 9], np.float32), 5, 1, 2) == [0, 2, 3, 5, 6]
    assert ref.choose(np.array([5, 3, 3, 3, 0, 2], np.float32), 3, 0, 1) == [0, 1, 5]
    assert ref.choose(np.zeros(2, np.float32), 4, 1, 1) == [0, 1, -1, -1]
