"""One token, one sequence, one head or no key head: dimensions of size 1, whose strides mean nothing. A single token laid out
heads first is contiguous, whatever its first stride says."""
import math

import pytest
import torch

from aegaeon_b200 import layout, ops

pytestmark = pytest.mark.gpu


def _odd_strides(t):
    """The same contiguous rows as ``t`` [1, heads, D] or [tokens, 1, D] with another stride on the axis of size 1."""
    out = torch.empty(t.size(1), t.size(0), t.size(2), dtype=t.dtype, device=t.device).transpose(0, 1)
    out.copy_(t)
    assert out.is_contiguous() and out.stride() != t.stride() and torch.equal(out, t)
    return out


def test_one_token_of_many_heads(cuda_device):
    g = torch.Generator(cuda_device).manual_seed(1)
    q, k, v = (torch.randn(1, n, 128, generator=g, device=cuda_device).half() for n in (8, 2, 2))
    pos, inv = torch.tensor([77], device=cuda_device), torch.rand(64, generator=g, device=cuda_device)
    want = ops.rotary_multi_axis(q, k, pos, inv, (64,))
    got = ops.rotary_multi_axis(_odd_strides(q), _odd_strides(k), pos, inv, (64,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = [_odd_strides(torch.zeros_like(x)) for x in (q, k)]
    ops.rotary_multi_axis(q, k, pos, inv, (64,), query_out=outs[0], key_out=outs[1])
    assert all(torch.equal(a, b) for a, b in zip(outs, want))

    caches = [torch.zeros(3, *layout.int4_block_shape(1, 2), dtype=torch.float16, device=cuda_device) for _ in range(2)]
    slot = torch.tensor([17], device=cuda_device)
    ops.reshape_and_cache_int4(k, v, caches[0], 0, slot)
    ops.reshape_and_cache_int4(_odd_strides(k), _odd_strides(v), caches[1], 0, slot)
    assert torch.equal(caches[0].view(torch.int16), caches[1].view(torch.int16))
    want = ops.gather_cache_int4(caches[0], 0, slot)
    got = ops.gather_cache_int4(caches[0], 0, slot, *(_odd_strides(torch.zeros_like(k)) for _ in range(2)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("planned", [False, True])
def test_one_sequence(cuda_device, planned):
    g = torch.Generator(cuda_device).manual_seed(2)
    q = torch.randn(1, 8, 128, generator=g, device=cuda_device).half()
    rows = torch.randn(2, 80, 2, 128, generator=g, device=cuda_device).half()
    cache = torch.zeros(6, *layout.int4_block_shape(1, 2), dtype=torch.float16, device=cuda_device)
    tables = torch.tensor([[4, 1, 0, 5, 2]], dtype=torch.int32, device=cuda_device)
    at = torch.arange(80, device=cuda_device)
    ops.reshape_and_cache_int4(rows[0], rows[1], cache, 0, tables[0].long()[at // 16] * 16 + at % 16)
    lens = torch.tensor([75], dtype=torch.int32, device=cuda_device)
    scale, want = 1 / math.sqrt(128), torch.empty_like(q)
    ops.paged_attention_decode_int4(want, q, cache, 0, tables, lens, scale)
    column = torch.empty(5, 1, dtype=torch.int32, device=cuda_device).T  # [1, 5] with strides (1, 1)
    column.copy_(tables)
    assert column.stride() == (1, 1) and column.is_contiguous()
    ops.read_device_errors(cuda_device)
    for t in (tables, column):
        plan = ops.DecodePlan(1, 8, 2, 128, cuda_device, cache="int4").plan(lens, t) if planned else None
        out = _odd_strides(torch.zeros_like(q))
        ops.paged_attention_decode_int4(out, _odd_strides(q), cache, 0, t, lens, scale, plan=plan)
        assert torch.equal(out, want)
    assert ops.read_device_errors(cuda_device) == 0


def test_one_head(cuda_device):
    g = torch.Generator(cuda_device).manual_seed(3)
    q, k = (torch.randn(5, 1, 128, generator=g, device=cuda_device).half() for _ in range(2))
    pos, inv = torch.arange(5, device=cuda_device), torch.rand(64, generator=g, device=cuda_device)
    want = ops.rotary_multi_axis(q, k, pos, inv, (64,))
    got = ops.rotary_multi_axis(_odd_strides(q), _odd_strides(k), pos, inv, (64,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    caches = [torch.zeros(3, *layout.int4_block_shape(1, 1), dtype=torch.float16, device=cuda_device) for _ in range(2)]
    for cache, x in zip(caches, (k, _odd_strides(k))):
        ops.reshape_and_cache_int4(x, x, cache, 0, pos + 3)
    assert torch.equal(caches[0].view(torch.int16), caches[1].view(torch.int16))


def test_queries_without_keys_and_positions_below_zero(cuda_device):
    g = torch.Generator(cuda_device).manual_seed(4)
    q = torch.randn(9, 4, 128, generator=g, device=cuda_device).half()
    pos, inv = torch.arange(-4, 5, device=cuda_device) * 1000, torch.rand(64, generator=g, device=cuda_device)
    want = ops.rotary_multi_axis(q, q, pos, inv, (64,))[0]
    got, none = ops.rotary_multi_axis(q, q[:, :0], pos, inv, (64,))
    assert torch.equal(got, want) and none.shape == (9, 0, 128)
    back, _ = ops.rotary_multi_axis(want, want, -pos, inv, (64,))
    # two roundings to fp16 of numbers that a rotation may mix with a partner of up to 5
    assert ((back.double() - q.double()).abs() <= 2 * 2.0 ** -11 * (q.double().abs() + 5)).all()
