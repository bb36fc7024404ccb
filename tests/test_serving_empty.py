"""Steps without rows and batches without sequences, by way of the C ABI and of the binding (CPU only: such calls launch
nothing)."""
import ctypes
import types

import pytest
import torch

from lucciola_rs_amd import library
from test_serving_abi import APPEND, APPEND4, ATTENTION, EXTEND, TRUNCATE, P, call


@pytest.fixture
def cdll():
    return library.load_cdll()


def test_arrays_of_no_rows_may_be_null(cdll):
    f = cdll.luc_block_extend
    none = dict(new=None, lens=None, tables=None, cu=None, start=None)
    assert call(f, EXTEND, batch=0, rows=0, slots=None, positions=None, **none) == 0
    assert call(f, EXTEND, batch=0, **none) == 0
    for name in ("free", "state"):
        assert call(f, EXTEND, batch=0, **{name: None}) == -1, name
    assert call(cdll.luc_block_truncate, TRUNCATE, batch=0, keep=None, lens=None, tables=None) == 0
    rows = ("q", "k", "v", "q_out", "positions", "slots")
    for fn, base in ((cdll.luc_kv4_append, APPEND4), (cdll.luc_qk_norm_rope_append, APPEND)):
        assert call(fn, base, rows=0, **dict.fromkeys(rows)) == 0
        for name in rows:
            assert call(fn, base, rows=0, **{name: None}) == 0
            assert call(fn, base, rows=1, **{name: None}) == -1
        for name in ("cos", "sin", "k_pool", "v_pool"):
            assert call(fn, base, rows=0, **{name: None}) == -1, name
        assert call(fn, base, rows=0, q=None, layer=2) == -1    # what is wrong stays so
    f = cdll.luc_kv4_attention
    assert call(f, ATTENTION, rows=0, q=None, out=None) == 0
    assert call(f, ATTENTION, batch=0, rows=0, q=None, out=None, cu=None, tables=None, start=None) == 0
    for name in ("tables", "start", "k_pool", "v_pool"):
        assert call(f, ATTENTION, rows=0, **{name: None}) == -1, name
    assert call(f, ATTENTION, batch=0, rows=9, q=None) == -1


@pytest.fixture
def lib():
    """A binding whose context no call reads, on CPU tensors."""
    lib = object.__new__(library.LucAttn)
    lib.lib, lib.ctx, lib.device = library.load_cdll(), P(1), -1
    yield lib
    lib.ctx = ctypes.c_void_p()  # (nothing to free)


def test_empty_tensors(lib):
    stream = types.SimpleNamespace(cuda_stream=0)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    assert half(0, 256).data_ptr() == 0
    lib.block_extend(i32(0), i32(0), i32(0, 4), i32(8), i32(4), i64(0), i32(0), i32(1), i32(0), stream=stream)
    lib.block_truncate(i32(0), i32(0), i32(0, 4), i32(8), i32(4), stream=stream)
    qkv = half(3, 8 * 64)[:0]
    cos = torch.zeros(10, 32)
    pool4, pool16 = torch.zeros(2, 1, 2, 640, dtype=torch.uint8), half(2, 1, 2, 16, 64)
    kw = dict(q=qkv[:, :256], k=qkv[:, 256:384], v=qkv[:, 384:], cos=cos, sin=cos, positions=i32(0), slots=i64(0),
              layer=0, num_layers=1, hq=4, hkv=2, head_dim=64, stream=stream)
    lib.kv4_append(**kw, k_pool=pool4, v_pool=pool4)
    lib.kv4_append(**kw, k_pool=pool4, v_pool=pool4, q_out=half(0, 256), k_out=half(0, 128), v_out=half(0, 128))
    lib.qk_norm_rope_append(**kw, k_pool=pool16, v_pool=pool16, q_out=half(0, 256), k_out=half(0, 128))
    for batch in (3, 0):
        lib.kv4_attention(half(0, 256), half(0, 256), pool4, pool4, i32(batch, 2), i32(batch), batch, 0, 0, 32, 0, 1, 4, 2,
                          64, 0.125, cu_seqlens=i32(batch + 1), stream=stream)
    # q of a padded step, none of whose rows is any sequence's
    lib.kv4_attention(half(0, 256), qkv[:, :256], pool4, pool4, i32(3, 2), i32(3), 3, 0, 1, 32, 0, 1, 4, 2, 64, 0.125,
                      cu_seqlens=i32(4), workspace=torch.zeros(64), stream=stream)
