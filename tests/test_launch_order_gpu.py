"""Early tile requests of a decode attention never pass a cache write further back than the kernel just
before it: two launches between the write and the attention's own wait, on a plan that was used before."""
import pytest
import torch

from aegaeon_b200 import layout, ops

pytestmark = pytest.mark.gpu

B, N_TOKENS, HQ, HKV = 32, 355, 8, 4
BLOCKS = (N_TOKENS + 15) // 16
SCALE = 128 ** -0.5


class Chain:
    """32 sequences of 355 tokens in a cache of two layers, and two sets of keys and values for them."""

    def __init__(self, dev, int4):
        g = torch.Generator(dev).manual_seed(5)
        pool = B * BLOCKS
        self.tables = torch.randperm(pool, generator=g, device=dev).to(torch.int32).view(B, BLOCKS)
        self.lens = torch.full((B,), N_TOKENS, dtype=torch.int32, device=dev)
        at = torch.arange(N_TOKENS, device=dev)
        self.slots = (self.tables.long()[:, at // 16] * 16 + at % 16).flatten()
        self.last = torch.arange(N_TOKENS - 1, B * N_TOKENS, N_TOKENS, device=dev)  # the newest token of each
        self.sets = [torch.randn(B * N_TOKENS, HKV, 128, generator=g, device=dev).half() for _ in range(2)]
        self.q = torch.randn(B, HQ, 128, generator=g, device=dev).half()
        shape = layout.int4_block_shape(2, HKV) if int4 else layout.kv_block_shape(2, HKV, 128)
        self.kv = torch.zeros((pool, *shape), dtype=torch.float16, device=dev)
        self.int4 = int4
        self.plan = ops.DecodePlan(B, HQ, HKV, 128, dev, cache="int4" if int4 else "auto").plan(self.lens, self.tables)
        self.inv = torch.ones(64, device=dev)
        self.pos = torch.arange(B, device=dev)

    def write(self, layer, x, slots):
        (ops.reshape_and_cache_int4 if self.int4 else ops.reshape_and_cache)(x, x, self.kv, layer, slots)

    def attend(self, **early):
        out = torch.empty_like(self.q)
        call = ops.paged_attention_decode_int4 if self.int4 else ops.paged_attention_decode
        call(out, self.q, self.kv, 0, self.tables, self.lens, SCALE, plan=self.plan, **early)
        return out

    def between(self, what, x):
        if what == "rotary":
            ops.rotary_multi_axis(self.q, self.q[:, :HKV], self.pos, self.inv, (64,))
        elif what == "write":
            self.write(1, x[self.last], self.slots[self.last])
        elif what == "read-back":
            ops.gather_cache_int4(self.kv, 1, self.slots[:64])
        elif what == "free":
            ops.free_blocks(self.lens.new_zeros(4), self.tables.new_zeros(2, 2), self.lens.new_zeros(2), self.pos[:1])


@pytest.mark.parametrize("int4,what", [(False, "rotary"), (False, "write"), (False, "free"), (True, "rotary"), (True, "write"),
                                       (True, "read-back"), (True, "free")])
def test_prefetch_two_launches_behind_a_write(cuda_device, int4, what):
    c = Chain(cuda_device, int4)
    want = []
    for x in c.sets:
        c.write(0, x, c.slots)
        torch.cuda.synchronize()
        want.append(c.attend())
    assert not torch.equal(*want)
    got = []
    for i in range(40):
        x = c.sets[i % 2]
        c.write(0, x, c.slots)
        c.between(what, x)
        got.append(c.attend(prefetch=True))
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(got))
    assert ops.read_device_errors(cuda_device) == 0


def test_after_decode_write_behind_a_prompt_write(cuda_device):
    """All but the newest positions by one write, the newest by the write just before the attention."""
    c = Chain(cuda_device, False)
    want, parts = [], []
    old = torch.ones(B * N_TOKENS, dtype=torch.bool, device=cuda_device)
    old[c.last] = False
    for x in c.sets:
        c.write(0, x, c.slots)
        torch.cuda.synchronize()
        want.append(c.attend())
        parts.append((x[old], c.slots[old], x[c.last], c.slots[c.last]))
    got = []
    for i in range(40):
        prompt, prompt_slots, new, new_slots = parts[i % 2]
        c.write(0, prompt, prompt_slots)
        c.write(0, new, new_slots)
        got.append(c.attend(after_decode_write=True))
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(got))


@pytest.mark.parametrize("int4", [False, True])
def test_captured_layers_with_a_write_before_each(cuda_device, int4):
    """The two-call layer in a graph: writes directly behind attentions let their successor start early."""
    c = Chain(cuda_device, int4)
    for x in c.sets:
        c.write(0, x, c.slots)
    c.write(1, c.sets[0], c.slots)
    new = [x[c.last].clone() for x in c.sets]
    at = c.slots[c.last]
    outs = [torch.empty_like(c.q) for _ in range(2)]
    call = ops.paged_attention_decode_int4 if int4 else ops.paged_attention_decode
    early = {} if int4 else dict(after_decode_write=True)

    def step():
        for layer in range(2):
            c.write(layer, new[layer], at)
            call(outs[layer], c.q, c.kv, layer, c.tables, c.lens, SCALE, plan=c.plan, **early)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(cuda_device).manual_seed(8)
    for _ in range(10):
        for x in new:
            x.copy_(torch.randn(x.shape, generator=g, device=cuda_device))
        graph.replay()
        got = [o.clone() for o in outs]
        for layer in range(2):  # the same, one call at a time
            c.write(layer, new[layer], at)
            torch.cuda.synchronize()
            call(outs[layer], c.q, c.kv, layer, c.tables, c.lens, SCALE, plan=c.plan)
            assert torch.equal(outs[layer], got[layer])
