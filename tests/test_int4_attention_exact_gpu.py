"""Decode attention over a 4-bit cache whose values lie far apart, against the oracle in 64 bits: poisoned groups
beside finite ones, and scores too large for a difference of rounded products."""
import pytest
import torch

from aegaeon_b200 import ops
from oracle import serving_ref as ref
from tests.test_int4_attention_gpu import SCALE, _bound, _cache, _q, _run

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


def _pairs(cache):
    """(blocks, layers, heads, key/value, token, group, scale/minimum) of a CPU cache, a view."""
    N, L, Hkv, _ = cache.shape
    return cache[..., 1024:].view(N, L, Hkv, 2, 16, 2, 2)


def _check(dev, q, cache, tables, lens, bound):
    """The finite outputs within ``bound``, NaN where the oracle has it."""
    ops.read_device_errors(dev)
    got = _run(dev, q, cache, 0, tables, lens, SCALE).double()
    assert ops.read_device_errors(dev) == 0
    want = ref.attention(q, cache, 0, tables, lens, SCALE)
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(got), bad)
    off = ((got - want).abs() / bound(want, q, cache, 0, tables, lens, SCALE))[~bad]
    assert (off <= 1).all(), f"off by {off.max():.3f} of the bound"


@BOTH
@pytest.mark.parametrize("size", [0.3, 1.0, 300.0])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_poisoned_group_leaves_the_other_group_alone(cuda_device, dtype, size, where):
    """More pairs than worker warps, so that a unit is a sequence's 19 tiles of a head; one tile of half of the
    heads has a value group without a finite span. The head's other 64 dims are finite and right."""
    lens, Hkv = [300, 289, 300], 640
    cache = _cache(dtype, 19, 1, Hkv, 6)
    pairs = _pairs(cache)
    pairs[:, :, :, 1] *= size
    block = {"first": 0, "middle": 9, "last": 18}[where]
    pairs[block, 0, ::4, 1, 0, 0] = float("nan")  # token 0 of the tile, dims 0..63
    pairs[block, 0, 1::4, 1, 0, 1] = float("nan")  # dims 64..127
    tables = torch.arange(19, dtype=torch.int32).repeat(3, 1).numpy()
    _check(cuda_device, _q(dtype, 3, Hkv), cache, tables, lens, _bound)


@BOTH
@pytest.mark.parametrize("size,sign", [(2.0 ** 10, 1), (2.0 ** 14, 1), (2.0 ** 14, -1), (1e17, 1), (1e17, -1)])
def test_scores_of_any_size_pick_the_largest(cuda_device, dtype, size, sign):
    """Queries and keys that are constant over their dims: scores of +-2^24 to 2^120 in log2 units, the largest
    ahead of the others by 10^6 and more. The output is that token's value row."""
    if size > 65504 and dtype == torch.float16:
        size = 2.0 ** 15
    for n in (3, 90, 250):
        cache = _cache(dtype, 16, 1, 2, n)
        pairs = _pairs(cache)
        best = n // 2
        steps = torch.randperm(256, generator=torch.Generator().manual_seed(n)) % 100
        steps[best] = 200
        unit = size * torch.finfo(dtype).eps if dtype == torch.float16 else size / 1024  # bf16: all but the best round alike
        pairs[:, 0, :, 0, :, :, 0] = 0
        pairs[:, 0, :, 0, :, :, 1] = (sign * (size + sign * unit * steps.float())).to(dtype).view(16, 1, 16, 1)
        q = torch.full((1, 8, 128), size, dtype=dtype)
        got = _run(cuda_device, q, cache, 0, torch.arange(16, dtype=torch.int32).view(1, 16).numpy(), [n])
        want = ref.values(cache[:, 0])[1][best // 16, :, best % 16].repeat_interleave(4, 0)
        # P * s with 11 bits times codes up to 8 off the middle; the scale is below 0.35, the minimum below 8
        bound = want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -11 * 8 * 0.35 + 2.0 ** -20 * 8
        assert ((got[0].double() - want).abs() <= bound).all()
