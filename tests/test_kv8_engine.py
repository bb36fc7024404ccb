"""Kv8Cache on the host, what it allocates, keeps and refuses (the library's sizes and a stand-in for its launches), and
calls without rows, which launch nothing (CPU only)."""
import ctypes
import types
import weakref

import pytest
import torch

from lucciola_rs_amd import library
from lucciola_rs_amd.engine import Kv8Cache
from test_kv8_abi import APPEND, ATTENTION, READ, SELECT, SPARSE, P, call


class Lib:
    """The host library's sizes; launches are only counted."""

    def __init__(self):
        host = library.load_cdll()
        self.lib = types.SimpleNamespace(luc_kv8_workspace_size=host.luc_kv8_workspace_size,
                                         luc_kv8_sparse_workspace_size=host.luc_kv8_sparse_workspace_size)
        self.calls = []

    def __getattr__(self, name):
        if name not in ("block_extend", "block_truncate", "kv8_append", "kv8_read", "kv8_attention", "kv8_select",
                        "kv8_sparse_attention"):
            raise AttributeError(name)
        return lambda *a, **kw: self.calls.append((name, a, kw))


@pytest.fixture
def capturing(monkeypatch):
    """[whether the current stream captures]"""
    flag = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: flag[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: None)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: None)
    return flag


def cache(hq=28, hkv=4, d=128, seqs=1, max_rows=1200, bounds=True):
    return Kv8Cache(1, hq, hkv, d, 4, seqs, 32768, max_rows, bounds, device="cpu", lib=Lib())


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (12, 2, 128), (14, 2, 64)])
def test_workspaces_that_nobody_holds_are_freed(capturing, hq, hkv, d):
    """Prompts of growing lengths, steps of growing contexts, dense and sparse: what stays allocated is a small
    multiple of the largest need, and zero-filled."""
    c = cache(hq, hkv, d)
    seen, largest = [], 0
    calls = [(rows, rows, 32 * rows - 16, None) for rows in range(1, 1000, 7)]
    calls += [(1, 1, ctx, budget) for ctx in range(16, 32769, 112) for budget in (None, 8, 96)]
    for rows, most, ctx, budget in calls:
        ws = c.workspace(rows, most, ctx, budget)
        need = c.lib.lib.luc_kv8_workspace_size(1, rows, most, ctx, hq, hkv, d) if budget is None else \
            c.lib.lib.luc_kv8_sparse_workspace_size(1, ctx, budget, hq, hkv, d)
        assert (ws is None) == (need == 0)
        if ws is not None:
            if not seen or seen[-1]() is not ws:
                seen.append(weakref.ref(ws))
            assert ws.numel() * 4 >= need and not bool(ws[:65536].any())
            largest = max(largest, need)
        del ws
    assert largest > 0
    alive = sum(w().numel() * 4 for w in seen if w() is not None)
    assert alive <= 1.5 * largest + 4 and len(seen) < 20


def test_workspaces_of_captures_are_kept(capturing):
    c = cache()
    small = weakref.ref(c.workspace(1, 1, 4000))
    capturing[0] = True
    assert c.workspace(1, 1, 4000) is small()
    with pytest.raises(RuntimeError, match="Kv8Cache.*before the capture"):
        c.workspace(1000, 1000, 32768)
    with pytest.raises(RuntimeError, match="before the capture"):
        c.workspace(1, 1, 1 << 20, 2000)
    capturing[0] = False
    eager = weakref.ref(c.workspace(700, 700, 32768))
    last = c.workspace(1100, 1100, 32768)
    assert small() is not None and (eager() is None or eager() is last)  # a graph has the one, nobody the other
    capturing[0] = True
    for _ in range(3):
        assert c.workspace(1100, 1100, 32768) is last and c.workspace(1, 1, 30000, 50) is last
    assert [w is x for w, x in zip(c._captured, (small(), last))] == [True, True] and len(c._captured) == 2


def test_calls_of_a_step(capturing):
    """An append of more rows than the step has is refused; attend and attend_sparse take one workspace."""
    c = cache(4, 2, 64, seqs=2, max_rows=10)
    rope = types.SimpleNamespace(cos=None, sin=None)
    new = torch.zeros(2, dtype=torch.int32)
    q = [torch.zeros(n, 256) for n in range(11)]
    for rows, most in ((8, 8), (2, 2), (0, 0), (None, 10)):
        c.extend(new, rows=rows)
        c.lib.calls.clear()
        for n in range(11):
            if n > most:
                with pytest.raises(ValueError, match=f"{n} rows to append: the step has {most}"):
                    c.append(0, q[n], q[n], q[n], rope)
            else:
                c.append(0, q[n], q[n], q[n], rope)
        assert len(c.lib.calls) == most + 1
    c.lib.calls.clear()
    pages = c.attend_sparse(0, q[2], q[2], 32768, 40, first=3)
    c.attend(0, q[2], q[2], 32768, max_rows=1)
    (select, a, kw), (attend, b, kb), (dense, _, kd) = c.lib.calls
    assert (select, attend, dense) == ("kv8_select", "kv8_sparse_attention", "kv8_attention")
    assert a[0] is pages and b[7] is pages and pages.shape == (2, 2, 40) and pages.dtype is torch.int32
    assert a[8:10] == (3, 2)
    assert kw["workspace"] is kb["workspace"] is not None and kd["workspace"] is not None
    own = torch.zeros(2, 2, 7, dtype=torch.int32)
    assert c.attend_sparse(0, q[2], q[2], 32768, 7, pages=own) is own
    without = cache(4, 2, 64, seqs=2, bounds=False)
    assert without.bounds is None
    with pytest.raises(ValueError, match="bounds=True"):
        without.attend_sparse(0, q[2], q[2], 32768, 40)


def test_arrays_of_no_rows_may_be_null():
    c = library.load_cdll()
    rows = ("q", "k", "v", "q_out", "positions", "slots")
    assert call(c.luc_kv8_append, APPEND, rows=0, **dict.fromkeys(rows)) == 0
    for name in rows:
        assert call(c.luc_kv8_append, APPEND, rows=0, **{name: None}) == 0
        assert call(c.luc_kv8_append, APPEND, rows=1, **{name: None}) == -1
    for name in ("cos", "sin", "k_pool", "v_pool", "scales"):
        assert call(c.luc_kv8_append, APPEND, rows=0, **{name: None}) == -1, name
    assert call(c.luc_kv8_append, APPEND, rows=0, q=None, layer=2) == -1    # what is wrong stays so
    assert call(c.luc_kv8_read, READ, rows=0, k_out=None, v_out=None, slots=None) == 0
    for name in ("k_pool", "v_pool", "scales"):
        assert call(c.luc_kv8_read, READ, rows=0, **{name: None}) == -1, name
    none = dict(cu=None, tables=None, start=None)
    for fn, base in ((c.luc_kv8_attention, ATTENTION), (c.luc_kv8_sparse_attention, SPARSE)):
        assert call(fn, base, rows=0, q=None, out=None) == 0
        assert call(fn, base, batch=0, rows=0, q=None, out=None, **none) == 0
        for name in ("tables", "start", "k_pool", "v_pool", "scales"):
            assert call(fn, base, rows=0, **{name: None}) == -1, name
        assert call(fn, base, batch=0, rows=9, q=None) == -1
    assert call(c.luc_kv8_sparse_attention, SPARSE, batch=0, rows=0, pages=None) == 0
    assert call(c.luc_kv8_select, SELECT, batch=0, rows=0, q=None, pages=None, **none) == 0
    for name in ("pages", "tables", "start", "bounds", "scales"):
        assert call(c.luc_kv8_select, SELECT, rows=0, **{name: None}) == -1, name


def test_empty_tensors():
    lib = object.__new__(library.LucAttn)
    lib.lib, lib.ctx, lib.device = library.load_cdll(), P(1), -1
    try:
        stream = types.SimpleNamespace(cuda_stream=0)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
        half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
        slots, qkv, cos = torch.zeros(0, dtype=torch.int64), half(3, 8 * 64)[:0], torch.zeros(10, 32)
        pool, scales = torch.zeros(2, 1, 2, 1024, dtype=torch.uint8), torch.zeros(2, 1, 2, 2)
        bounds = torch.zeros(2, 1, 2, 2, 64, dtype=torch.uint8)
        lib.kv8_append(qkv[:, :256], qkv[:, 256:384], qkv[:, 384:], cos, cos, i32(0), slots, pool, pool, scales, 0, 1, 4, 2,
                       64, bounds=bounds, q_out=half(0, 256), stream=stream)
        lib.kv8_read(half(0, 128), half(0, 128), slots, pool, pool, scales, 0, 1, 2, 64, stream=stream)
        for batch in (3, 0):
            lib.kv8_attention(half(0, 256), half(0, 256), pool, pool, scales, i32(batch, 2), i32(batch), batch, 0, 0, 32, 0,
                              1, 4, 2, 64, 0.125, cu_seqlens=i32(batch + 1), stream=stream)
            lib.kv8_sparse_attention(half(0, 256), half(0, 256), pool, pool, scales, i32(batch, 2), i32(batch),
                                     i32(batch, 2, 3), batch, 32, 0, 1, 4, 2, 64, 0.125, cu_seqlens=i32(batch + 1),
                                     stream=stream)
        lib.kv8_select(i32(0, 2, 3), half(0, 256), bounds, scales, i32(0, 2), i32(0), 0, 32, 1, 2, 0, 1, 4, 2, 64,
                       cu_seqlens=i32(1), stream=stream)
    finally:
        lib.ctx = ctypes.c_void_p()  # (nothing to free)
