"""The new operators as a server uses them together: prompts with image positions go into a 4-bit cache,
requests are forked into parallel samples, decode steps rotate, write and attend, samples are dropped,
the pool is compacted and decoding goes on. Checked against one oracle that keeps every sequence's cache
rows by itself, without blocks."""
import math

import pytest
import torch

from aegaeon_b200 import layout, ops
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu

SECTIONS = (16, 24, 24)


class Oracle:
    """Each sequence's quantised rows in a small cache of its own (blocks in order)."""

    def __init__(self, dtype, L, Hkv, inv):
        self.dtype, self.L, self.Hkv, self.inv, self.seqs = dtype, L, Hkv, inv, {}

    def fork(self, a, b):
        self.seqs[b] = (self.seqs[a][0].clone(), self.seqs[a][1])

    def append(self, row, layer, key, value):
        cache, n = self.seqs.setdefault(row, (torch.zeros(12, *layout.int4_block_shape(self.L, self.Hkv), dtype=self.dtype), 0))
        ref.write(cache, layer, key, value, range(n, n + key.size(0)))
        if layer == self.L - 1:
            self.seqs[row] = (cache, n + key.size(0))

    def attend(self, row, layer, q, n):
        return ref.attention(q.unsqueeze(0), self.seqs[row][0], layer, [list(range(12))], [n], 1 / math.sqrt(128))[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_forks_steps_and_compaction(cuda_device, dtype):
    dev, L, Hq, Hkv, N, R, W = cuda_device, 2, 8, 2, 64, 8, 12
    g = torch.Generator().manual_seed(9)
    inv = (1.0 / 1e6 ** (torch.arange(64) / 64)).float()
    oracle = Oracle(dtype, L, Hkv, inv)
    kv = torch.zeros(N, *layout.int4_block_shape(L, Hkv), dtype=dtype, device=dev)
    counts, lens = torch.zeros(N, dtype=torch.int32, device=dev), torch.zeros(R, dtype=torch.int32, device=dev)
    tables, free = torch.zeros(R, W, dtype=torch.int32, device=dev), torch.randperm(N, generator=g).tolist()
    inv_dev = inv.to(dev)
    ops.read_device_errors(dev)

    def rows(n, heads):
        return torch.randn(n, heads, 128, generator=g).to(dtype)

    # Prompts of three requests, an image of 4 x 5 patches in each.
    prompts = {0: 37, 1: 64, 2: 5 + 20}
    pos, slots = [], []
    for r, n in prompts.items():
        t = torch.arange(n)
        image = (t >= 3) & (t < 23)
        p = torch.stack([torch.where(image, torch.tensor(3), t), torch.where(image, 3 + (t - 3) // 5, t), torch.where(image, 3 + (t - 3) % 5, t)])
        pos.append(p)
        table = [free.pop() for _ in range((n + 15) // 16)]
        tables[r, :len(table)] = torch.tensor(table, dtype=torch.int32)
        counts[table] = 1
        slots += layout.slots_for(table, 0, n)
    lens[:3] = torch.tensor(list(prompts.values()), dtype=torch.int32)
    pos, slots = torch.cat(pos, 1), torch.tensor(slots)
    for layer in range(L):
        q, k, v = rows(len(slots), Hq), rows(len(slots), Hkv), rows(len(slots), Hkv)
        _, dk = ops.rotary_multi_axis(q.to(dev), k.to(dev), pos.to(dev), inv_dev, SECTIONS)
        ops.reshape_and_cache_int4(dk, v.to(dev), kv, layer, slots.to(dev))
        # the oracle takes the rotated keys as the kernel rounded them; the rotation has its own test
        at = 0
        for r, n in prompts.items():
            oracle.append(r, layer, dk[at:at + n].cpu(), v[at:at + n])
            at += n

    def grow(live):
        """The next token's block where a row begins a new one (the server's block manager)."""
        updates = []
        for r in live:
            n = int(lens[r])
            if n % 16 == 0:
                b = int((counts == 0).nonzero()[0])
                counts[b] = 1
                updates.append((r, n // 16, b))
        ops.update_block_tables(tables, updates)

    def step(live):
        grow(live)
        idx = torch.tensor(live, device=dev)
        before = lens[idx]
        lens[idx] += 1
        step_tables, step_lens = tables[idx].contiguous(), lens[idx].contiguous()
        inp = ops.prepare_step_inputs(step_tables, before.contiguous(), step_lens)
        plan = ops.DecodePlan(len(live), Hq, Hkv, 128, dev, cache="int4").plan(step_lens, step_tables)
        for layer in range(L):
            q, k, v = rows(len(live), Hq), rows(len(live), Hkv), rows(len(live), Hkv)
            dq, dk = ops.rotary_multi_axis(q.to(dev), k.to(dev), inp.positions.expand(3, -1), inv_dev, SECTIONS)
            ops.reshape_and_cache_int4(dk, v.to(dev), kv, layer, inp.slot_mapping)
            out = torch.empty_like(dq)
            ops.paged_attention_decode_int4(out, dq, kv, layer, step_tables, step_lens, 1 / math.sqrt(128), plan=plan)
            for i, r in enumerate(live):
                n = oracle.seqs[r][1] + 1
                oracle.append(r, layer, dk[i:i + 1].cpu(), v[i:i + 1])
                want = oracle.attend(r, layer, dq[i].cpu(), n)
                # bounds as in test_int4_attention_gpu.py, for scales below 1/2 and outputs below 4: half a
                # step of the output and 2^-11 * 8 * 0.5 for the rounded products, the rest far below
                bound = want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -11 * 8 * 0.5 + 2.0 ** -12
                assert ((out[i].cpu().double() - want).abs() <= bound).all()
        assert ops.read_device_errors(dev) == 0

    step([0, 1, 2])
    assert ops.fork_blocks(kv, counts, tables, lens, [0, 0, 1, 2], [3, 4, 5, 6]).numel() == 4
    for a, b in ((0, 3), (0, 4), (1, 5), (2, 6)):
        oracle.fork(a, b)
    for _ in range(3):
        step([0, 1, 2, 3, 4, 5, 6])
    ops.free_blocks(counts, tables, lens, [0, 5])
    ops.fork_blocks(kv, counts, tables, lens, [3], [7])
    oracle.fork(3, 7)
    got = ops.compact_blocks(kv, counts, tables, lens)
    live = int(got.num_live)
    assert live == int((counts > 0).sum()) and not got.ref_counts[live:].any()
    counts, tables = got.ref_counts, got.block_tables
    kv[live:] = float("nan")  # the tail now belongs to someone else
    for _ in range(9):
        step([1, 2, 3, 4, 6, 7])
    ops.free_blocks(counts, tables, lens, list(range(R)))
    assert not counts.any() and not lens.any() and ops.read_device_errors(dev) == 0
