"""Workspace sizes of attention over the quantised caches at the largest sizes that the calls allow: a plan of
its splits, or a refusal, and never the end of the process (CPU only)."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ASK = """
import sys
import __graft_entry__
__graft_entry__.load_package()
from lucciola_rs_amd import library
fn = getattr(library.load_cdll(), sys.argv[1])
for line in sys.argv[2:]:
    print(fn(*map(int, line.split(","))))
"""


def sizes(fn, *calls):
    """fn of each call's arguments, in a process of its own."""
    lines = [",".join(map(str, c)) for c in calls]
    done = subprocess.run([sys.executable, "-c", ASK, fn, *lines], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    return [int(x) for x in done.stdout.split()]


# batch, total_rows, max_rows, max_ctx, q heads, kv heads, head_dim: so many workgroups of one context each that their rounds alone
# ask for more than 2^31 tokens a split, or a little less
LARGEST = [(n, n, 1, 1 << 30, h, h, d) for n, h, d in (
    (65536, 1, 64), (65536, 1, 128), (49152, 1, 64), (32768, 1, 128), (4096, 1, 64), (8192, 8, 128), (2048, 8, 64), (4096, 4, 64))]
LARGEST += [(8192, 8192, 1, 1 << 26, 64, 8, 128), (16384, 16384, 2, 1 << 29, 8, 2, 64)]


@pytest.mark.parametrize("fn", ["luc_kv8_workspace_size", "luc_kv4_workspace_size"])
def test_the_largest_calls_have_a_plan(fn):
    """One split of every context: no workspace."""
    assert sizes(fn, *LARGEST) == [0] * len(LARGEST)


@pytest.mark.parametrize("fn", ["luc_kv8_workspace_size", "luc_kv4_workspace_size"])
def test_long_contexts_keep_their_splits(fn):
    """Of two splits or more, each has partials of 8 columns: (m, l) and o, behind 2^16 counters."""
    for size, (batch, splits, d) in zip(sizes(fn, (1, 1, 1, 1 << 30, 8, 1, 64), (2, 2, 1, 1 << 30, 8, 1, 128)),
                                        ((1, 256, 64), (2, 256, 128))):
        assert size == (1 << 18) + batch * splits * 8 * (8 + 4 * d)


def test_the_largest_choices_have_a_plan():
    got = sizes("luc_kv8_sparse_workspace_size", (65536, 1 << 30, 1 << 26, 1, 1, 64), (65536, 1 << 30, 1 << 25, 1, 1, 64),
                (8192, 1 << 30, 1 << 26, 64, 8, 128))
    # fewer pages than a context's need room for their scores; the attention has one split of each
    assert got == [0, (1 << 18) + 65536 * (1 << 26) * 4, 0]
