"""luc_block_extend and luc_block_truncate against the one-page-at-a-time form and the host allocator."""
import numpy as np
import pytest
import torch

import serving_ref as ref
from lucciola_rs_amd.engine import BlockManager

pytestmark = pytest.mark.gpu
PAGE = 16


class Device:
    def __init__(self, luc, batch, stride, num_blocks):
        i32 = dict(dtype=torch.int32, device="cuda")
        self.luc, self.batch = luc, batch
        self.lens = torch.zeros(batch, **i32)
        self.tables = torch.zeros(batch, stride, **i32)
        self.free = torch.arange(num_blocks - 1, -1, -1, **i32)
        self.state = torch.zeros(4, **i32)
        self.state[0] = num_blocks
        self.cu = torch.full((batch + 1,), 77, **i32)
        self.start = torch.full((batch,), 77, **i32)

    def extend(self, new, rows):
        slots = torch.full((rows,), 99, dtype=torch.int64, device="cuda")
        positions = torch.full((rows,), 99, dtype=torch.int32, device="cuda")
        n = torch.tensor(new, dtype=torch.int32, device="cuda")
        self.luc.block_extend(n, self.lens, self.tables, self.free, self.state, slots, positions,
                              self.cu, self.start)
        return slots.tolist(), positions.tolist(), self.cu.tolist(), self.start.tolist()

    def truncate(self, keep):
        k = torch.tensor(keep, dtype=torch.int32, device="cuda")
        self.luc.block_truncate(k, self.lens, self.tables, self.free, self.state)

    def everything(self):
        count = int(self.state[0])
        return (self.lens.tolist(), self.tables.tolist(), self.free[:count].tolist(), self.state[1:].tolist())


def same(dev, maps):
    lens, tables, free, rest = dev.everything()
    assert lens == maps.lens
    assert np.array_equal(np.array(tables, np.int32), maps.tables)
    assert free == maps.free
    assert rest == [0, 0, 0]


@pytest.mark.parametrize("batch,most", [(1, 1), (1, 40), (2, 17), (7, 1), (33, 100), (64, 700), (300, 33),
                                        (1025, 20), (4096, 3)])
def test_steps_against_one_page_at_a_time(luc, batch, most):
    """Ragged growth (zeros among it), roll-backs and releases, over several workgroups too."""
    rng = np.random.default_rng(batch + most)
    stride = 4 * most // PAGE + 3
    blocks = batch * stride
    dev, maps = Device(luc, batch, stride, blocks), ref.Maps(batch, stride, blocks)
    for step in range(5):
        new = rng.integers(0, most + 1, batch)
        if step == 1:
            new[:] = 1
        if step == 3:
            new[:] = 0
        new = [min(int(n), stride * PAGE - maps.lens[b]) for b, n in enumerate(new)]
        rows = sum(new) + (0, 5, 2100)[step % 3]
        print(f"  batch {batch} step {step}: {sum(new)} new rows of {rows}", flush=True)
        slots, positions, cu, start = dev.extend(new, rows)
        ws, wp, wc, wst = maps.extend(new)
        pad = [-1] * (rows - len(ws))
        assert slots == ws + pad and positions == wp + pad
        assert cu == wc and start == wst
        same(dev, maps)
        keep = [int(rng.integers(0, n + 3)) if rng.random() < 0.5 else n for n in maps.lens]
        dev.truncate(keep)
        maps.truncate(keep)
        same(dev, maps)


def test_undone_step_restores_everything(luc):
    dev = Device(luc, 9, 40, 300)
    dev.extend([3, 100, 0, 16, 17, 50, 1, 1, 33], 400)
    dev.truncate([3, 30, 0, 0, 17, 50, 1, 0, 16])
    before, free = dev.everything(), dev.free.tolist()
    lens = dev.lens.tolist()
    dev.extend([40, 0, 16, 1, 15, 200, 31, 5, 0], 400)
    dev.truncate(lens)
    assert dev.everything() == before and dev.free.tolist() == free


def test_same_pages_as_the_host_allocator(luc):
    rng = np.random.default_rng(3)
    batch, stride, blocks = 6, 12, 60
    dev, host = Device(luc, batch, stride, blocks), BlockManager(blocks, batch, stride)
    lens = [0] * batch
    for _ in range(30):
        b = int(rng.integers(batch))
        if rng.random() < 0.3:
            dev.truncate([0 if i == b else 10 ** 6 for i in range(batch)])
            host.release(b)
            lens[b] = 0
        else:
            n = int(rng.integers(0, min(60, stride * PAGE - lens[b]) + 1))
            if host.num_free < -(-(lens[b] + n) // PAGE) - host.num_pages(b):
                continue
            dev.extend([n if i == b else 0 for i in range(batch)], 64)
            lens[b] += n
            host.reserve(b, lens[b])
        assert dev.lens.tolist() == lens
        assert np.array_equal(dev.tables.cpu().numpy(), host.table())
        assert int(dev.state[0]) == host.num_free
    host.close()


@pytest.mark.parametrize("case", ["pages", "table", "negative", "rows", "state", "lens", "both", "rows and pages"])
def test_refused_extends_change_nothing(luc, case):
    dev = Device(luc, 4, 5, 12)
    dev.extend([20, 30, 1, 0], 60)
    rows, new, bits = 4000, [1, 1, 1, 1], 0
    if case == "pages":
        new, bits = [40, 40, 40, 40], 1  # 5 pages are held, 8 of 7 are asked for
    elif case == "table":
        new, bits = [1, 51, 0, 0], 2
    elif case == "negative":
        new, bits = [1, -1, 1, 1], 4
    elif case == "rows":
        rows, new, bits = 3, [1, 1, 1, 1], 8
    elif case == "state":
        dev.state[0], bits = 13, 4
    elif case == "lens":
        dev.lens[2], bits = 81, 4
    elif case == "both":
        # lengths 80 and 80 take 3 + 3 pages more, of 7 free: the rows alone are short
        rows, new, bits = 10, [60, 50, 0, 0], 8
    elif case == "rows and pages":
        rows, new, bits = 10, [60, 50, 16, 16], 1 | 8  # 3 + 3 + 1 + 1 pages
    lens, tables, free, _ = dev.everything()
    slots, positions, cu, start = dev.extend(new, rows)
    assert slots == [-1] * rows and positions == [-1] * rows and cu == [0] * 5
    assert start == lens
    assert dev.everything() == (lens, tables, free, [bits, 0, 0])
    # the status stays, later calls work
    if case not in ("state", "lens"):
        assert dev.extend([1, 0, 0, 0], 8)[0][0] >= 0
        assert dev.state[1].item() == bits


def test_refused_truncates_change_nothing(luc):
    dev = Device(luc, 3, 5, 12)
    dev.extend([20, 30, 1], 60)
    before = dev.everything()
    dev.truncate([0, -1, 0])
    assert dev.everything() == (*before[:3], [4, 0, 0])
    dev.state[1] = 0
    dev.state[0] = 10  # with 10 pages free, the 5 held are more than the pool has
    dev.truncate([0, 0, 0])
    assert dev.lens.tolist() == before[0] and dev.state.tolist() == [10, 4, 0, 0]


def test_pages_outside_the_pool_are_no_slots(luc):
    dev = Device(luc, 2, 8, 16)
    # handed out: 0, 1, 2, 3 from the end of the list 15, ..., 0; the first and third damaged
    dev.free[15], dev.free[13] = 16, -3
    slots, positions, _, _ = dev.extend([17, 18], 40)
    assert slots[:16] == [-1] * 16 and slots[16] == 1 * 16
    assert slots[17:33] == [-1] * 16 and slots[33] == 3 * 16
    assert positions[:35] == list(range(17)) + list(range(18))
    # neither is a held entry that was damaged later
    dev.tables[0, 1] = 1 << 30
    assert dev.extend([2, 0], 8)[0][:2] == [-1, -1]


def test_captured_steps_on_another_stream(luc):
    """A captured step (extend by one, every third replay a roll-back of two) against the plain form."""
    batch, stride, blocks = 5, 10, 64
    dev, maps = Device(luc, batch, stride, blocks), ref.Maps(batch, stride, blocks)
    new = torch.tensor([1, 1, 0, 1, 1], dtype=torch.int32, device="cuda")
    keep = torch.full((batch,), 10 ** 6, dtype=torch.int32, device="cuda")
    slots = torch.zeros(8, dtype=torch.int64, device="cuda")
    positions = torch.zeros(8, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        luc.block_truncate(keep, dev.lens, dev.tables, dev.free, dev.state)
        luc.block_extend(new, dev.lens, dev.tables, dev.free, dev.state, slots, positions, dev.cu, dev.start)
    for i in range(40):
        want = [max(0, n - 2) for n in maps.lens] if i % 3 == 2 else [10 ** 6] * batch
        keep.copy_(torch.tensor(want, dtype=torch.int32))
        graph.replay()
        maps.truncate(want)
        ws, wp, wc, wst = maps.extend([1, 1, 0, 1, 1])
        torch.cuda.synchronize()
        assert slots.tolist() == ws + [-1] * 4 and positions.tolist() == wp + [-1] * 4
        assert dev.cu.tolist() == wc and dev.start.tolist() == wst
        same(dev, maps)
