"""Decode attention over a 4-bit cache whose values lie far apart, against the oracle in 64 bits: poisoned groups
beside finite ones, scores too large for a difference of rounded products, tokens and groups whose scales differ
by many powers of two, query elements far below the head's largest.

Tolerance (``_weighted``), from the exact weights w, scales s, minima m and values V of each token, for a
sequence of n tokens (t tiles of 16):
  * the output's own rounding: half a step of its value;
  * w * s is kept to 16 bits, times codes of up to 15: 2^-16 * 15 * sum w s;
  * two products a tile on the tensor cores, each cut off by up to 2^-22 of what the sum holds, at most
    15 * sum w s: 2 t * 2^-22 of that; the sums of w m in fp32, (t + 8) * 2^-23 * sum w (|m| + 15 s);
  * a score is off by 2^-22 for each of its 8 products and 8 more steps, of the sum of its absolute terms, A,
    and by 2^-23 of itself in the exponent; a weight moves by twice that and by 2^-21 for its exponential and
    the sum that divides it, the output by as much of sum w |V| and of itself."""
import pytest
import torch

from aegaeon_b200 import ops
from oracle import serving_ref as ref
from tests.gpu_helpers import make_tables
from tests.test_int4_attention_gpu import SCALE, _bound, _cache, _q, _run

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


def _pairs(cache):
    """(blocks, layers, heads, key/value, token, group, scale/minimum) of a CPU cache, a view."""
    N, L, Hkv, _ = cache.shape
    return cache[..., 1024:].view(N, L, Hkv, 2, 16, 2, 2)


def _weighted(want, q, cache, layer, tables, lens, scale):
    """The tolerance above, per output element. In fp16 keys' codes count with an offset of 64."""
    B, Hq, _ = q.shape
    Hkv = cache.size(2)
    out = torch.empty_like(want)
    for b in range(B):
        n = int(lens[b])
        tiles = (n + 15) // 16
        ids = torch.as_tensor([int(i) for i in tables[b][:tiles]])
        k, v = (x.transpose(0, 1).reshape(Hkv, -1, 128)[:, :n] for x in ref.values(cache[ids, 0]))
        pairs = _pairs(cache)[ids, 0].double().permute(1, 2, 0, 3, 4, 5).reshape(Hkv, 2, -1, 2, 2)[:, :, :n]
        qg = q[b].double().view(Hkv, -1, 128)
        w = torch.softmax(torch.einsum("hgd,htd->hgt", qg, k) * scale, -1)
        sk, mk = (pairs[:, 0, :, :, i].repeat_interleave(64, -1) for i in (0, 1))  # Hkv, n, 128
        size = 2 * 79 * sk + mk.abs() if q.dtype == torch.float16 else (k - mk).abs() + mk.abs()  # 64 + c, 64 s beside m
        terms = torch.einsum("hgd,htd->hgt", qg.abs(), size)
        delta = (16 * 2.0 ** -22 + 2.0 ** -23) * terms.amax(-1) * abs(scale) * 1.5  # Hkv, G, in log2 units
        sv, mv = (pairs[:, 1, :, :, i].repeat_interleave(64, -1).nan_to_num() for i in (0, 1))
        ws = torch.einsum("hgt,htd->hgd", w, sv)
        wm = torch.einsum("hgt,htd->hgd", w, mv.abs() + 15 * sv)
        wv = torch.einsum("hgt,htd->hgd", w, v.abs().nan_to_num())
        err = 15 * ws * (2.0 ** -16 + 2 * tiles * 2.0 ** -22) + wm * (tiles + 8) * 2.0 ** -23
        err = err + (2 * delta.unsqueeze(-1) + 2.0 ** -21) * 2 * wv
        out[b] = err.reshape(Hq, 128)
    info = torch.finfo(q.dtype)
    return out + want.abs() * info.eps / 2 + info.smallest_normal * info.eps


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
        # P * s with 16 bits times codes up to 15; the scale is below 0.35, the minimum below 8
        bound = want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -16 * 15 * 0.35 + 2.0 ** -20 * 8
        assert ((got[0].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,large,small", [(torch.float16, 8000.0, 2.0 ** -12), (torch.bfloat16, 1e9, 0.3),
                                               (torch.bfloat16, 1e20, 1e-3), (torch.bfloat16, 3.0, 1e-20)])
def test_a_large_scale_without_weight_costs_the_others_nothing(cuda_device, dtype, large, small):
    """One token's value scale is 2^24 times the others' and more, and no query looks at it."""
    cache = _cache(dtype, 8, 1, 2, 6)
    pairs = _pairs(cache)
    g = torch.Generator().manual_seed(2)
    pairs[..., 1, :, :, 0] = (small * (0.5 + torch.rand(8, 1, 2, 16, 2, generator=g))).to(dtype)
    pairs[..., 1, :, :, 1] = (-7.5 * pairs[..., 1, :, :, 0].float()).to(dtype)
    pairs[3, 0, :, 1, 5, :, 0] = large
    pairs[3, 0, :, 1, 5, :, 1] = -7.5 * large
    pairs[3, 0, :, 0, 5, :, 0] = 0.0
    pairs[3, 0, :, 0, 5, :, 1] = -40.0  # its score lies 200 and more below the others
    q = (_q(dtype, 1, 8).abs() + 0.5).to(dtype)
    tables = torch.arange(8, dtype=torch.int32).view(1, 8).numpy()
    _check(cuda_device, q, cache, tables, [128], _weighted)


@pytest.mark.parametrize("dtype,ratio", [(torch.float16, 2.0 ** 26), (torch.bfloat16, 2.0 ** 26), (torch.bfloat16, 2.0 ** 60)])
@pytest.mark.parametrize("lens", [[128, 33, 7], [300, 289, 300]])
def test_groups_of_one_head_with_scales_far_apart(cuda_device, dtype, ratio, lens):
    """The values of dims 64..127 are 2^26 or 2^60 times smaller than those of dims 0..63."""
    Hkv = 2 if lens[0] < 300 else 640  # units of one tile, and of whole sequences
    N = sum((n + 15) // 16 for n in lens)
    cache = _cache(dtype, N, 1, Hkv, 4)
    pairs = _pairs(cache)
    high = 2.0 ** 12 if dtype == torch.float16 else 2.0 ** 20
    pairs[..., 1, :, 0, :] *= high
    pairs[..., 1, :, 1, :] *= high / ratio
    _check(cuda_device, _q(dtype, 3, Hkv), cache, make_tables(lens, N, 3), lens, _weighted)


@BOTH
def test_outputs_carry_their_types_precision(cuda_device, dtype):
    """Ordinary values, to the outputs' own rounding: few tokens, where each one's weight is large."""
    lens = [1, 5, 17, 40, 100, 333]
    N = sum((n + 15) // 16 for n in lens)
    _check(cuda_device, _q(dtype, 6, 8), _cache(dtype, N, 1, 2, 4), make_tables(lens, N, 3), lens, _weighted)


def test_small_elements_of_a_bf16_query_count_in_full(cuda_device):
    """Dim 0 holds the query's largest element and the keys' zeros; the scores come from elements 2^-20 times
    as large and keys of up to 10^6."""
    dtype, n = torch.bfloat16, 60
    cache = _cache(dtype, 4, 1, 1, 9)
    raw = cache.view(torch.uint8).view(4, 1, 1, 2304)
    raw[..., torch.arange(16) * 64] &= 0xf0  # key dim 0: code 0
    pairs = _pairs(cache)
    g = torch.Generator().manual_seed(5)
    pairs[:, :, :, 0, :, :, 0] = (1e5 * (0.5 + torch.rand(4, 1, 1, 16, 2, generator=g))).to(dtype)
    pairs[:, :, :, 0, :, :, 1] = 0
    q = (torch.randn(1, 8, 128, generator=g) * 2.0 ** -20).to(dtype)
    q[..., 0] = 1.0
    _check(cuda_device, q, cache, torch.arange(4, dtype=torch.int32).view(1, 4).numpy(), [n], _weighted)


@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e30, 2e38])
def test_bf16_queries_of_any_size(cuda_device, size):
    """Scores of ordinary size from queries near either end of bf16's range; the keys' scales make up for it."""
    dtype, lens = torch.bfloat16, [70, 16, 1, 300]
    cache = _cache(dtype, 27, 1, 2, 9)
    pairs = _pairs(cache)
    pairs[:, :, :, 0] = (pairs[:, :, :, 0].double() / size).clamp(-3e38, 3e38).to(dtype)
    q = (_q(dtype, 4, 8).double().clamp(-1.6, 1.6) * size).to(dtype)
    _check(cuda_device, q, cache, make_tables(lens, 27, 3), lens, _weighted)


def test_a_plan_for_rows_laid_out_otherwise_is_refused(cuda_device):
    """Tables that begin at the same address and are as wide, their rows further apart: other blocks."""
    wide = torch.arange(16, dtype=torch.int32, device=cuda_device).view(2, 8)
    near, far = wide.flatten()[:8].view(2, 4), wide[:, :4]
    assert near.data_ptr() == far.data_ptr() and near.shape == far.shape
    lens = torch.tensor([60, 64], dtype=torch.int32, device=cuda_device)
    cache, q = _cache(torch.float16, 16, 1, 2, 3).to(cuda_device), _q(torch.float16, 2, 4).to(cuda_device)
    kv = torch.zeros(16, 1, 2, 16, 2, 128, dtype=torch.float16, device=cuda_device)
    for kind, call, pool in (("int4", ops.paged_attention_decode_int4, cache), ("auto", ops.paged_attention_decode, kv)):
        plan = ops.DecodePlan(2, 4, 2, 128, cuda_device, cache=kind).plan(lens, near)
        call(torch.empty_like(q), q, pool, 0, near, lens, SCALE, plan=plan)
        call(torch.empty_like(q), q, pool, 0, wide.flatten()[:8].view(2, 4), lens, SCALE, plan=plan)
        with pytest.raises(ValueError, match="plan"):
            call(torch.empty_like(q), q, pool, 0, far, lens, SCALE, plan=plan)


# ---- wide groups, shared workspaces -----------------------------------------------------------------


@BOTH
@pytest.mark.parametrize("G", [9, 16])
def test_groups_of_more_than_eight_heads(cuda_device, dtype, G):
    """Two column tiles: ordinary values to the outputs' precision, scales 2^26 apart between the groups, and a
    poisoned group in units of 19 tiles (more pairs than the 1036 workers)."""
    lens = [1, 17, 333]
    N = sum((n + 15) // 16 for n in lens)
    cache, tables = _cache(dtype, N, 1, 2, 4), make_tables(lens, N, 3)
    _check(cuda_device, _q(dtype, 3, 2 * G), cache, tables, lens, _weighted)
    pairs = _pairs(cache)
    pairs[..., 1, :, 0, :] *= 2.0 ** 12
    pairs[..., 1, :, 1, :] *= 2.0 ** -14
    _check(cuda_device, _q(dtype, 3, 2 * G), cache, tables, lens, _weighted)
    lens, Hkv = [300, 289, 300], 400
    cache = _cache(dtype, 19, 1, Hkv, 6)
    _pairs(cache)[0, 0, ::4, 1, 0, 0] = float("nan")
    _pairs(cache)[9, 0, 1::4, 1, 0, 1] = float("nan")
    tables = torch.arange(19, dtype=torch.int32).repeat(3, 1).numpy()
    _check(cuda_device, _q(dtype, 3, Hkv * G), cache, tables, lens, _weighted)


def test_two_captured_graphs_share_a_workspace(cuda_device):
    """One plan's step in two graphs, each with its own queries and layers, replayed in any order."""
    dtype, N, lens = torch.float16, 260, [3000, 40, 0, 177, 16]
    cache, tables = _cache(dtype, N, 3, 2, 12).to(cuda_device), torch.as_tensor(make_tables(lens, N, 5)).to(cuda_device)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    plan = ops.DecodePlan(5, 14, 2, 128, cuda_device, cache="int4")
    qs = [_q(dtype, 5, 14, i).to(cuda_device) for i in range(2)]
    outs = [[torch.empty_like(qs[0]) for _ in range(3)] for _ in range(2)]

    def step(i):
        plan.plan(sl, tables)
        for layer in range(3):
            ops.paged_attention_decode_int4(outs[i][layer], qs[i], cache, layer, tables, sl, SCALE, plan=plan, prefetch=layer > 0)

    want, graphs = [], []
    for i in range(2):
        step(i)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs[i]])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            step(i)
    for i in (0, 1, 1, 0, 0, 1):
        for o in outs[i]:
            o.fill_(7)
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    assert ops.read_device_errors(cuda_device) == 0
