"""The 4-bit cache's write and read-back, bit for bit against the oracle."""
import pytest
import torch

from aegaeon_b200 import layout, ops
from aegaeon_b200._native import AEG_DEVERR_SLOT_RANGE
from oracle import serving_ref as ref
from tests.test_serving_ref_cpu import _hard_rows

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


def _bits(t):
    return t.contiguous().view(torch.int16).cpu()


def _same_but_nan(a, b):
    """Equal bits, any NaN for a NaN."""
    a, b = a.cpu(), b.cpu()
    nan = torch.isnan(b)
    assert torch.equal(torch.isnan(a), nan)
    assert torch.equal(torch.where(nan, 0, a), torch.where(nan, 0, b))


def _run(dev, dtype, N, L, Hkv, layer, key, value, slots):
    g = torch.Generator().manual_seed(N)
    start = torch.randint(-32768, 32768, (N, *layout.int4_block_shape(L, Hkv)), generator=g).to(torch.int16).view(dtype)
    cache = start.to(dev)
    ops.reshape_and_cache_int4(key.to(dev), value.to(dev), cache, layer, slots.to(dev))
    want = start.clone()
    ref.write(want, layer, key, value, slots)
    return cache, want


@BOTH
@pytest.mark.parametrize("T,Hkv", [(1, 1), (1, 40), (7, 4), (37, 3), (300, 8), (2500, 4), (5000, 5)])
def test_write_changes_the_named_rows_alone(cuda_device, dtype, T, Hkv):
    g = torch.Generator().manual_seed(T)
    N = T // 16 + 9
    key = (torch.randn(T, Hkv, 128, generator=g) * 3 + torch.randn(128, generator=g)).to(dtype)
    value = torch.randn(T, Hkv, 128, generator=g).to(dtype)
    slots = torch.randperm(N * 16, generator=g)[:T]
    if T > 20:
        slots[3], slots[10] = -1, -12345
    ops.read_device_errors(cuda_device)
    cache, want = _run(cuda_device, dtype, N, 3, Hkv, 1, key, value, slots)
    assert torch.equal(_bits(cache), _bits(want))
    assert ops.read_device_errors(cuda_device) == 0
    k, v = ops.gather_cache_int4(cache, 1, slots.to(cuda_device))
    for got, x in zip((k, v), ref.gather(want, 1, slots)):
        assert torch.equal(_bits(got), _bits(x))


@BOTH
def test_ties_subnormals_offsets_and_wide_spreads(cuda_device, dtype):
    rows = _hard_rows(dtype, 6000, torch.Generator().manual_seed(11))
    n = rows.size(0) // 2 * 2
    x = rows[:n].view(-1, 1, 128)
    T = x.size(0)
    slots = torch.arange(T)
    cache, want = _run(cuda_device, dtype, T // 16 + 1, 1, 1, 0, x, x.flip(0), slots)
    finite = _bits(want).view(-1, 1152)
    got = _bits(cache).view(-1, 1152)
    assert torch.equal(got[:, :1024], finite[:, :1024])
    _same_but_nan(cache.view(-1, 1152)[:, 1024:], want.view(-1, 1152)[:, 1024:])


@BOTH
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_group_without_a_finite_span_reads_back_as_nan(cuda_device, dtype, bad):
    key = torch.randn(4, 2, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    value = key.flip(0).contiguous()
    key[1, 0, 70] = bad
    value[2, 1, 5] = bad
    slots = torch.tensor([0, 17, 18, 40])
    cache, want = _run(cuda_device, dtype, 3, 1, 2, 0, key, value, slots)
    k, v = ops.gather_cache_int4(cache, 0, slots.to(cuda_device))
    expect_k = torch.zeros(4, 2, 128, dtype=torch.bool)
    expect_k[1, 0, 64:] = True
    expect_v = torch.zeros(4, 2, 128, dtype=torch.bool)
    expect_v[2, 1, :64] = True
    assert torch.equal(torch.isnan(k).cpu(), expect_k) and torch.equal(torch.isnan(v).cpu(), expect_v)
    for got, x in zip((k, v), ref.gather(want, 0, slots)):
        _same_but_nan(got, x)


def test_largest_bf16_values(cuda_device):
    top = torch.finfo(torch.bfloat16).max
    x = torch.full((2, 1, 128), 0.0)
    x[0, 0, :64] = top / 2
    x[0, 0, 3] = -top / 2  # a span of the largest value itself
    x[1, 0, 0], x[1, 0, 1] = top, -top  # beyond fp32
    x = x.to(torch.bfloat16)
    slots = torch.tensor([0, 1])
    cache, want = _run(cuda_device, torch.bfloat16, 1, 1, 1, 0, x, x, slots)
    k, _ = ops.gather_cache_int4(cache, 0, slots.to(cuda_device))
    assert torch.isfinite(k[0]).all() and torch.isnan(k[1, 0, :64]).all() and not torch.isnan(k[1, 0, 64:]).any()
    _same_but_nan(k, ref.gather(want, 0, slots)[0])


@BOTH
def test_strided_and_unaligned_rows(cuda_device, dtype):
    T, Hq, Hkv = 33, 6, 2
    qkv = torch.randn(T, (Hq + 2 * Hkv) * 128 + 1, generator=torch.Generator().manual_seed(2)).to(dtype)
    dev = qkv.to(cuda_device)
    slots = torch.arange(T)
    for off in (0, 1, 3):  # off 1 and the odd token stride take the 2-byte path
        key, value = (qkv[:, off + a:off + a + Hkv * 128].view(T, Hkv, 128) for a in (0, 2 * 128))
        dkey, dvalue = (dev[:, off + a:off + a + Hkv * 128].view(T, Hkv, 128) for a in (0, 2 * 128))
        cache = torch.zeros(3, 1, Hkv, 1152, dtype=dtype, device=cuda_device)
        ops.reshape_and_cache_int4(dkey, dvalue, cache, 0, slots.to(cuda_device))
        want = torch.zeros(3, 1, Hkv, 1152, dtype=dtype)
        ref.write(want, 0, key, value, slots)
        assert torch.equal(_bits(cache), _bits(want))
        out = torch.zeros_like(dev)
        ok, ov = (out[:, off + a:off + a + Hkv * 128].view(T, Hkv, 128) for a in (0, 2 * 128))
        ops.gather_cache_int4(cache, 0, slots.to(cuda_device), ok, ov)
        for got, x in zip((ok, ov), ref.gather(want, 0, slots)):
            assert torch.equal(_bits(got), _bits(x))


@BOTH
def test_slots_outside_are_skipped_and_reported(cuda_device, dtype):
    ops.read_device_errors(cuda_device)
    x = torch.randn(3, 1, 128).to(dtype)
    cache, want = _run(cuda_device, dtype, 2, 1, 1, 0, x, x, torch.tensor([5, 32, -1]))
    assert torch.equal(_bits(cache), _bits(want))
    assert ops.read_device_errors(cuda_device) == AEG_DEVERR_SLOT_RANGE
    k, v = ops.gather_cache_int4(cache, 0, torch.tensor([1 << 40, -3, 5], device=cuda_device))
    assert not k[:2].any() and not v[:2].any()
    assert torch.equal(_bits(k[2]), _bits(ref.gather(want, 0, [5])[0][0]))
    assert ops.read_device_errors(cuda_device) == AEG_DEVERR_SLOT_RANGE


def test_empty_calls_and_refusals(cuda_device):
    cache = torch.zeros(2, 1, 4, 1152, dtype=torch.float16, device=cuda_device)
    none = torch.empty(0, 4, 128, dtype=torch.float16, device=cuda_device)
    no_slots = torch.empty(0, dtype=torch.int64, device=cuda_device)
    ops.reshape_and_cache_int4(none, none, cache, 0, no_slots)
    assert ops.gather_cache_int4(cache, 0, no_slots)[0].shape == (0, 4, 128)
    row = torch.zeros(1, 4, 128, dtype=torch.float16, device=cuda_device)
    slot = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    for bad in (dict(key=None), dict(key=row.bfloat16()), dict(key=row[:, :2]), dict(slots=slot.int()), dict(slots=slot.cpu()), dict(layer=1),
                dict(cache=cache[..., :1024]), dict(cache=cache.float()), dict(key=row.double()), dict(slots=slot.repeat(2))):
        a = dict(dict(key=row, cache=cache, layer=0, slots=slot), **bad)
        with pytest.raises(ValueError):
            ops.reshape_and_cache_int4(a["key"], a["key"], a["cache"], a["layer"], a["slots"])
    with pytest.raises(ValueError, match="together"):
        ops.gather_cache_int4(cache, 0, slot, key=row)
    with pytest.raises(NotImplementedError):
        half = torch.zeros(1, 4, 64, dtype=torch.float16, device=cuda_device)
        ops.reshape_and_cache_int4(half, half, cache, 0, slot)


def test_blocks_of_a_4bit_cache_move_like_any_others(cuda_device):
    cache = torch.randint(-32768, 32768, (6, 2, 4, 1152), dtype=torch.int32).to(torch.int16).view(torch.bfloat16).to(cuda_device)
    start = cache.clone()
    host = torch.empty(2, 2, 4, 1152, dtype=torch.bfloat16).pin_memory()
    ops.copy_blocks([0, 2], [1, 5], cache)
    ops.swap([1, 4], [1, 0], False, cache, host)
    ops.swap([0], [3], True, cache, host)
    torch.cuda.synchronize()
    want = start.clone()
    want[1], want[5], want[3] = start[0], start[2], start[4]
    assert torch.equal(_bits(cache), _bits(want)) and torch.equal(_bits(host[1]), _bits(start[0]))


def test_captured_write_replays_on_new_inputs(cuda_device):
    dtype = torch.bfloat16
    key = torch.randn(20, 2, 128, device=cuda_device).to(dtype)
    value = torch.randn(20, 2, 128, device=cuda_device).to(dtype)
    slots = torch.arange(20, device=cuda_device)
    cache = torch.zeros(4, 1, 2, 1152, dtype=dtype, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.reshape_and_cache_int4(key, value, cache, 0, slots)
            k, v = ops.gather_cache_int4(cache, 0, slots)
    torch.cuda.synchronize()
    key.copy_(torch.randn(20, 2, 128))
    slots.add_(30)
    graph.replay()
    torch.cuda.synchronize()
    want = torch.zeros(4, 1, 2, 1152, dtype=dtype)
    ref.write(want, 0, key.cpu(), value.cpu(), slots.cpu())
    assert torch.equal(_bits(cache), _bits(want))
    assert torch.equal(_bits(k), _bits(ref.gather(want, 0, slots.cpu())[0]))
