"""luc_kv8_append of rows in any order: a page's rows anywhere in the call are one run, as the plain form has it; and its q bit for
bit."""
import numpy as np
import pytest
import torch

from test_gpu_kv8_append import Book, PAGE, seq

pytestmark = pytest.mark.gpu


def packed(pages, lengths, starts, seed):
    """(slots, positions) of sequences one after the other, on pages in shuffled order."""
    perm = np.random.default_rng(seed).permutation(pages).tolist()
    s, p = [], []
    for n, start in zip(lengths, starts):
        need = -(-(start + n) // PAGE)
        x = seq(perm[:need], start, n)
        perm = perm[need:]
        s, p = s + x[0], p + x[1]
    return np.array(s), np.array(p)


def append(book, slots, pos, *scales):
    book.append([int(x) for x in slots], [int(x) for x in pos], book.rows(len(slots), *scales))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, "bf16"), (12, 2, 128, "f16")])
@pytest.mark.parametrize("seqs,tokens", [(64, 2), (33, 2), (40, 5), (64, 8), (200, 3), (65, 16), (300, 4)])
def test_token_by_token(luc, hq, hkv, d, dtype, seqs, tokens):
    """Every sequence's first row, then every one's second, and so on: at the beginnings of pages, over their ends, and
    louder into pages that hold tokens."""
    book = Book(luc, hq, hkv, d, dtype, pages=2 * seqs + 3, seed=seqs)
    for start, k_scale in ((0, 1.4), (tokens, 6.0), (2 * tokens, 0.1)):
        if start + tokens > 2 * PAGE:
            break
        s, p = packed(book.pages, [tokens] * seqs, [start] * seqs, 3)
        order = np.arange(seqs * tokens).reshape(seqs, tokens).T.reshape(-1)
        append(book, s[order], p[order], k_scale, 2.0)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, "f16"), (5, 1, 128, "bf16")])
@pytest.mark.parametrize("rows", [64, 65, 127, 300, 512, 513, 1100, 2500])
def test_any_order(luc, hq, hkv, d, dtype, rows):
    """Prompts, whole pages and ends of pages, as they come, their rows backwards, and in no order at all; with rows that have no
    place or no position among them, some of which name a slot of the call."""
    rng = np.random.default_rng(rows)
    cuts = np.sort(rng.choice(np.arange(1, rows), 3, replace=False))
    lengths = np.diff(np.concatenate([[0], cuts, [rows]]))
    starts = [0, 5, 16, 31]
    book = Book(luc, hq, hkv, d, dtype, pages=rows // PAGE + 14, seed=rows, norm=False)
    for i in range(3):
        s, p = packed(book.pages, lengths, starts, i)
        p = p % 400
        order = (np.arange(rows), np.arange(rows)[::-1], rng.permutation(rows))[i]
        s, p = s[order].copy(), p[order].copy()
        for at in rng.choice(rows, rows // 20, replace=False):
            if rng.integers(2):
                s[at] = (-1, 1 << 40, book.pages * PAGE)[rng.integers(3)]
            else:
                p[at] = (-1, 400, 1 << 30)[rng.integers(3)]
                s[at] = s[rng.integers(rows)]
        append(book, s, p, (1.4, 20.0, 0.3)[i], (1.0, 0.2, 5.0)[i])


@pytest.mark.parametrize("rows", [200, 700, 3000])
def test_the_ends_of_a_call(luc, rows):
    """A page of a call's first and last row, of rows 31, 32 and 33 apart, and one whose rows but one are side by side."""
    book = Book(luc, 4, 2, 64, "bf16", pages=rows // PAGE + 12, seed=rows)
    s, p = packed(book.pages - 6, [rows], [0], 1)
    p = p % 400
    extra = [(book.pages - 1, [(0, 3), (rows - 1, 4)]), (book.pages - 2, [(40, 0), (71, 1), (103, 2), (136, 3)]),
             (book.pages - 3, [(80 + i, i) for i in range(15)] + [(rows - 7, 15)]),
             (book.pages - 4, [(10, 15)] + [(160 + i, i) for i in range(15)]),
             (book.pages - 5, [(5, 7), (6, 8), (38, 9), (rows - 3, 1)])]
    for page, places in extra:
        for at, off in places:
            s[at] = page * PAGE + off
    append(book, s, p)
    append(book, s, p, 9.0, 0.1)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 64, "bf16"), (28, 4, 128, "f16")])
@pytest.mark.parametrize("rows", [5, 600])
def test_bits_of_q(luc, hq, hkv, d, dtype, rows):
    """q is that of luc_qk_norm_rope_append in every bit, zeros' signs too, and what lies behind a row stays."""
    book = Book(luc, hq, hkv, d, dtype, pages=rows // PAGE + 4, bias=False, seed=rows)
    a, b = hq * d, (hq + hkv) * d
    qkv = book.rows(rows)
    qkv[::3, :a:2] = 0.0
    qkv[1::3, :a:3] = -0.0
    qkv[2::5, :a] *= -0.0
    s, p = packed(book.pages, [rows], [0], 0)
    slots = torch.from_numpy(s).cuda()
    pos = torch.from_numpy(np.where(np.arange(rows) % 7 == 4, -1, p % 400).astype(np.int32)).cuda()
    kp, vp = (torch.zeros((book.pages, 2, hkv, PAGE, d), dtype=book.dt, device="cuda") for _ in range(2))
    want, got = (torch.full((rows, a + 8), 7.0, dtype=book.dt, device="cuda") for _ in range(2))
    args = (qkv[:, :a], qkv[:, a:b], qkv[:, b:], book.cos, book.sin, pos, slots)
    luc.qk_norm_rope_append(*args, kp, vp, 1, 2, hq, hkv, d, q_out=want[:, :a], **book.kw)
    luc.kv8_append(*args, book.k, book.v, book.scales, 1, 2, hq, hkv, d, bounds=book.bounds, q_out=got[:, :a], **book.kw)
    torch.cuda.synchronize()
    assert bool((want[:, :a].view(torch.int16) == -32768).any()) and bool((want[:, :a].view(torch.int16) == 0).any())
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
