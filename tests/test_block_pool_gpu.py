"""Forking, freeing and compacting shared blocks: everything equal to the oracle's lists."""
import random

import pytest
import torch

from aegaeon_b200 import ops
from aegaeon_b200._native import AEG_DEVERR_BLOCK_ID_RANGE, AEG_DEVERR_POOL_EMPTY, AEG_DEVERR_POOL_ENTRY
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu

BITS = {"entry": AEG_DEVERR_POOL_ENTRY, "empty": AEG_DEVERR_POOL_EMPTY, "id": AEG_DEVERR_BLOCK_ID_RANGE}


class Both:
    """The same pool on the device and in the oracle."""

    def __init__(self, dev, N, R, W, shape=(2, 2, 16, 1, 8), seed=0):
        r = random.Random(seed)
        self.dev, self.r = dev, r
        blocks = torch.randint(-32768, 32768, (N, *shape), dtype=torch.int32).to(torch.int16)
        tables = [[r.randrange(N) if N else 0 for _ in range(W)] for _ in range(R)]
        self.o = ref.Pool([0] * N, tables, [0] * R, blocks)
        self.kv = blocks.to(dev)
        self.sync_in()

    def fill(self, rows, lens):
        """Rows of their own blocks, spread over the pool."""
        free = [b for b, c in enumerate(self.o.counts) if c == 0]
        self.r.shuffle(free)
        for row, n in zip(rows, lens):
            for j in range((n + 15) // 16):
                b = free.pop()
                self.o.tables[row][j] = b
                self.o.counts[b] = 1
            self.o.lens[row] = n
        self.sync_in()

    def sync_in(self):
        i32 = dict(dtype=torch.int32, device=self.dev)
        self.counts, self.lens = torch.tensor(self.o.counts, **i32), torch.tensor(self.o.lens, **i32)
        self.tables = torch.tensor(self.o.tables, **i32).view(len(self.o.lens), -1)
        ops.read_device_errors(self.dev)

    def check(self, errors=()):
        assert ops.read_device_errors(self.dev) == sum(BITS[e] for e in errors)
        assert self.counts.tolist() == self.o.counts
        assert self.lens.tolist() == self.o.lens
        assert self.tables.tolist() == self.o.tables
        assert torch.equal(self.kv.cpu(), self.o.blocks)

    def fork(self, src, dst):
        new, errors = self.o.fork(src, dst)
        got = ops.fork_blocks(self.kv, self.counts, self.tables, self.lens, src, dst)
        assert got.tolist() == new
        self.check(errors)

    def free(self, rows):
        errors = self.o.free(rows)
        ops.free_blocks(self.counts, self.tables, self.lens, rows)
        self.check(errors)

    def compact(self, errors=()):
        tables, counts, remap, n = self.o.compact()
        before = [t.clone() for t in (self.counts, self.tables, self.lens)]
        got = ops.compact_blocks(self.kv, self.counts, self.tables, self.lens)
        for a, b in zip((self.counts, self.tables, self.lens), before):
            assert torch.equal(a, b)
        assert got.num_live.tolist() == [n] and got.remap.tolist() == remap
        assert got.ref_counts.tolist() == counts and got.block_tables.tolist() == tables
        self.check(errors)
        self.o.tables, self.o.counts = tables, counts
        self.counts, self.tables = got.ref_counts, got.block_tables


@pytest.mark.parametrize("N,R,W,shape", [(64, 10, 5, (2, 2, 16, 1, 8)), (5000, 40, 9, (1, 3)), (300, 60, 3, (5,)),
                                         (40, 12, 4, (28, 2, 16, 4, 128)), (90, 20, 4, (9, 1, 1152))])
def test_forks_frees_and_compactions_in_turn(cuda_device, N, R, W, shape):
    b = Both(cuda_device, N, R, W, shape, seed=N)
    half = R // 2
    lens = [b.r.choice([1, 15, 16, 17, 16 * W, b.r.randint(1, 16 * W)]) for _ in range(half)]
    while sum((n + 15) // 16 for n in lens) > N - half:
        lens[b.r.randrange(half)] = b.r.randint(0, 16)
    b.fill(range(half), lens)
    for _ in range(3):
        dst = [i for i in range(R) if b.o.lens[i] == 0]
        b.fork([b.r.randrange(half) for _ in dst], dst)
        b.free(b.r.sample(range(half, R), R // 4))
        b.compact()
    b.free(list(range(R)))
    assert b.o.counts == [0] * N
    b.compact()


def test_forks_of_forks_share_and_copy_the_tail(cuda_device):
    b = Both(cuda_device, 20, 6, 3)
    b.fill([0, 1], [33, 32])
    b.fork([0, 1, 0, 1], [2, 3, 4, 5])
    assert b.o.lens == [33, 32, 33, 32, 33, 32]
    shared, tail = b.o.tables[0][:2], b.o.tables[0][2]
    assert [b.o.counts[x] for x in shared] == [3, 3] and b.o.counts[tail] == 1
    b.free([0])
    b.free([2, 4])
    assert b.o.counts[shared[0]] == 0


def test_refused_entries_leave_their_rows_alone(cuda_device):
    b = Both(cuda_device, 12, 8, 3)
    b.fill([0, 1], [17, 5])
    # outside the table, onto a full row, onto one's own row, the same target twice, an empty source
    b.fork([0, 9, 0, 0, 1, 1, 6, -1], [2, 3, 1, 0, 2, 3, 4, 5])
    assert b.o.lens == [17, 5, 17, 5, 0, 0, 0, 0]
    # a target of this call as another entry's source: read as it was before, empty
    b.fork([0, 4, 1], [4, 5, 6])
    assert b.o.lens == [17, 5, 17, 5, 17, 0, 5, 0]
    b.free([0, 0, 5, 8, -1])
    b.free([2, 4, 1, 3, 6])
    assert b.o.counts == [0] * 12


def test_a_pool_that_runs_out_serves_the_first_entries(cuda_device):
    b = Both(cuda_device, 4, 9, 2)
    b.fill([0, 1], [3, 16])
    b.fork([0, 0, 1, 0, 0, 1], [2, 3, 4, 5, 6, 7])
    assert b.o.lens == [3, 16, 3, 3, 16, 0, 0, 16, 0]


def test_ids_outside_the_pool_are_reported(cuda_device):
    b = Both(cuda_device, 6, 5, 3)
    b.fill([0, 1], [40, 20])
    b.o.tables[0][1] = 77      # a full block
    b.o.tables[1][1] = -2      # the block a fork would copy
    b.sync_in()
    b.fork([0, 1], [2, 3])
    b.compact(("id",))
    b.free([0, 2])


def test_sharing_a_free_block_is_reported(cuda_device):
    b = Both(cuda_device, 8, 4, 2)
    b.fill([0], [32])
    b.o.counts[b.o.tables[0][0]] = 0
    b.sync_in()
    ops.fork_blocks(b.kv, b.counts, b.tables, b.lens, [0], [1])
    b.o.fork([0], [1])
    b.check(("entry",))


def test_more_forks_than_one_pass_over_the_entries(cuda_device):
    R = 2600
    b = Both(cuda_device, 4000, R, 2, (3,))
    b.fill(range(50), [b.r.choice([7, 16, 20, 32]) for _ in range(50)])
    dst = list(range(50, R))
    b.r.shuffle(dst)
    dst[10] = dst[2000]
    b.fork([b.r.randrange(50) for _ in dst], dst)
    b.free(dst[::3])
    b.compact()


@pytest.mark.parametrize("live", [0, 1, 7, 4095, 4096, 9000])
def test_compaction_at_the_edges(cuda_device, live):
    b = Both(cuda_device, 9000, 3, 3000, (2,))
    ids = b.r.sample(range(9000), live)
    for row in range(3):
        part = ids[3000 * row:3000 * (row + 1)]
        b.o.tables[row][:len(part)] = part
        b.o.lens[row] = 16 * len(part)
        for i in part:
            b.o.counts[i] = 1
    b.sync_in()
    b.compact()
    assert b.o.counts == [1] * live + [0] * (9000 - live)


def test_empty_pools_tables_and_calls(cuda_device):
    b = Both(cuda_device, 3, 2, 2)
    b.fork([], [])
    b.free([])
    kv = torch.empty(0, 4, device=cuda_device)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    got = ops.compact_blocks(kv, torch.empty(0, **i32), torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    assert got.num_live.tolist() == [0] and got.block_tables.tolist() == [[0, 0, 0], [0, 0, 0]]
    got = ops.compact_blocks(b.kv, b.counts, torch.zeros(0, 3, **i32), torch.zeros(0, **i32))
    assert got.num_live.tolist() == [0] and got.block_tables.shape == (0, 3)


def test_refusals(cuda_device):
    b = Both(cuda_device, 4, 3, 2)
    a = (b.kv, b.counts, b.tables, b.lens)
    with pytest.raises(ValueError, match="target rows"):
        ops.fork_blocks(*a, [0, 1], [2])
    for i, t in ((0, b.kv[:3]), (0, b.kv.cpu()), (1, b.counts.long()), (2, b.tables.view(-1)), (2, b.tables[:2]), (2, b.tables[:, :1]),
                 (3, b.lens[:2])):
        bad = list(a)
        bad[i] = t
        with pytest.raises(ValueError):
            ops.fork_blocks(*bad, [0], [1])
        with pytest.raises(ValueError):
            ops.compact_blocks(*bad)
        if i:
            with pytest.raises(ValueError):
                ops.free_blocks(*bad[1:], [0])


def test_a_captured_beam_step_replays(cuda_device):
    b = Both(cuda_device, 60, 9, 4)
    b.fill([0, 1, 2], [50, 33, 16])
    src = torch.tensor([0, 0, 1, 2, 1, 0], device=cuda_device)
    dst = torch.arange(3, 9, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.free_blocks(b.counts, b.tables, b.lens, dst)
            new = ops.fork_blocks(b.kv, b.counts, b.tables, b.lens, src, dst)
    torch.cuda.synchronize()
    for step in ([0, 0, 1, 2, 1, 0], [2, 2, 1, 1, 0, 0], [1, 1, 1, 1, 1, 1]):
        src.copy_(torch.tensor(step))
        graph.replay()
        torch.cuda.synchronize()
        b.o.free(list(range(3, 9)))
        want, _ = b.o.fork(step, list(range(3, 9)))
        assert new.tolist() == want
        b.check()


def test_copying_a_free_last_block_is_refused(cuda_device):
    """A row whose partly filled last block has no references: the lowest free block, which another entry takes."""
    b = Both(cuda_device, 8, 6, 2)
    b.fill([0, 1], [20, 5])
    tail = b.o.tables[0][1]
    b.o.counts[tail] = 0
    for block in range(tail):  # below it nothing is free
        b.o.counts[block] = max(b.o.counts[block], 1)
    b.sync_in()
    b.fork([0, 1, 0, 1], [2, 3, 4, 4])
    assert b.o.lens == [20, 5, 0, 5, 5, 0] and b.o.tables[3][0] == tail
