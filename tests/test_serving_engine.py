"""Kv4Cache on the host: what it allocates, keeps and refuses (CPU only, the library's sizes and a stand-in for its
launches)."""
import types
import weakref

import pytest
import torch

from lucciola_rs_amd import library
from lucciola_rs_amd.engine import Kv4Cache


class Lib:
    """The host library's sizes; launches are only counted."""

    def __init__(self):
        self.lib = types.SimpleNamespace(luc_kv4_workspace_size=library.load_cdll().luc_kv4_workspace_size)
        self.calls = []

    def __getattr__(self, name):
        if name not in ("block_extend", "block_truncate", "kv4_append", "kv4_attention"):
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


def cache(hq=28, hkv=4, d=128, seqs=1, max_rows=1200):
    return Kv4Cache(1, hq, hkv, d, 4, seqs, 32768, max_rows, device="cpu", lib=Lib())


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (12, 2, 128), (14, 2, 64)])
def test_workspaces_that_nobody_holds_are_freed(capturing, hq, hkv, d):
    """Prompts of growing lengths: what stays allocated is a small multiple of the largest need."""
    c = cache(hq, hkv, d)
    seen, largest = [], 0
    for rows in range(100, 1200):
        ws = c.workspace(rows, rows, rows)
        if ws is not None:
            if not seen or seen[-1]() is not ws:
                seen.append(weakref.ref(ws))
            need = c.lib.lib.luc_kv4_workspace_size(1, rows, rows, rows, hq, hkv, d)
            assert ws.numel() * 4 >= need and not bool(ws.any())
            largest = max(largest, need)
        del ws
    assert largest > 0
    alive = sum(w().numel() * 4 for w in seen if w() is not None)
    assert alive <= 1.5 * largest + 4 and len(seen) < 12
    # token steps up to a long context
    for ctx in range(16, 32769, 16):
        c.workspace(1, 1, ctx)
    assert sum(w() is not None for w in seen) <= 1


def test_workspaces_of_captures_are_kept(capturing):
    c = cache()
    small = weakref.ref(c.workspace(1, 1, 4000))
    capturing[0] = True
    assert c.workspace(1, 1, 4000) is small() and c.workspace(1, 1, 3000) is small()
    with pytest.raises(RuntimeError, match="before the capture"):
        c.workspace(1, 1, 32768)
    capturing[0] = False
    eager = weakref.ref(c.workspace(1, 1, 32768))
    last = c.workspace(1000, 1000, 32768)
    assert small() is not None and eager() is None     # a graph has the one, nobody the other
    assert c.workspace(1, 1, 100) in (None, last)
    capturing[0] = True
    for _ in range(3):
        assert c.workspace(1000, 1000, 32768) is last
    assert [w is x for w, x in zip(c._captured, (small(), last))] == [True, True] and len(c._captured) == 2


def test_an_append_of_more_rows_than_the_step_has(capturing):
    """Slots behind the last extend's rows are an earlier step's: such a row is refused."""
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
    with pytest.raises(ValueError, match="outside"):  # a step that is refused changes nothing
        c.extend(new, rows=11)
    c.append(0, q[10], q[10], q[10], rope)
