"""Decode attention over a 4-bit cache against the oracle in 64 bits.

Tolerance (``_bound``), for weights p that sum to 1, scales s and minima m as the cache holds them:
  * the output's own rounding: half a step of its value;
  * P * s rounded to fp16, 2^-11 of each term, times codes taken around their middle (|c - 8| <= 8):
    2^-11 * 8 * max s;
  * the sums of 16-token tiles on the tensor cores, each cut off by up to 2^-22 of what the sum holds:
    at most 32 tiles of (16 + 15) s before the constant is taken out, 8 s a tile of what stays;
  * the scores: 64 products a group of q with codes offset by up to 128, within 2^-19 of
    (143 s + |m|) * sum |q|, and 2^-22 of the score's own size for the exponent. Weights move by twice
    that, the output by as much of the values' spread."""
import math

import pytest
import torch

from aegaeon_b200 import layout, ops
from aegaeon_b200._native import (AEG_DEVERR_BLOCK_ID_RANGE, AEG_DEVERR_PLAN_MISMATCH, AEG_DEVERR_SEQ_LEN_RANGE)
from oracle import serving_ref as ref
from tests.gpu_helpers import make_tables

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
SCALE = 1.0 / math.sqrt(128)


def _bound(want, q, cache, layer, tables, lens, scale):
    B, Hq, _ = q.shape
    Hkv = cache.size(2)
    out = torch.empty_like(want)
    for b in range(B):
        n = max(int(lens[b]), 1)
        ids = torch.as_tensor([int(i) for i in tables[b][:(n + 15) // 16]])
        pairs = cache[ids, layer, :, 1024:].double().view(-1, Hkv, 2, 16, 2, 2).permute(1, 2, 0, 3, 4, 5).reshape(Hkv, 2, -1, 2, 2)
        pairs = pairs[:, :, :n].nan_to_num()
        s_k, m_k = pairs[:, 0, :, :, 0].amax(1), pairs[:, 0, :, :, 1].abs().amax(1)  # Hkv, group
        s_v, m_v = pairs[:, 1, :, :, 0].amax(1), pairs[:, 1, :, :, 1].abs().amax(1)
        qs = q[b].double().view(Hkv, -1, 2, 64).abs().sum(-1)
        score = ((143 * s_k + m_k).unsqueeze(1) * qs).sum(-1) * abs(scale)  # Hkv, G
        delta = 2.0 ** -19 * score + 2.0 ** -22 * (1 + score)
        spread = 15 * s_v + 2 * m_v
        tiles = (n + 15) // 16
        err = 2.0 ** -11 * 8 * s_v + 2.0 ** -22 * (32 * 31 + 8 * tiles) * s_v
        err = (2 * delta).unsqueeze(-1) * spread.unsqueeze(1) + err.unsqueeze(1)  # Hkv, G, group
        out[b] = err.repeat_interleave(64, -1).reshape(Hq, 128)
    info = torch.finfo(q.dtype)
    return out + want.abs() * info.eps / 2 + info.smallest_normal * info.eps


def _cache(dtype, N, L, Hkv, seed, kind="normal"):
    """A CPU cache of quantised random rows in every slot."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros(N, *layout.int4_block_shape(L, Hkv), dtype=dtype)
    raw = cache.view(torch.uint8).view(N, L, Hkv, 2304)
    raw[..., :2048] = torch.randint(0, 256, (N, L, Hkv, 2048), generator=g).to(torch.uint8)
    pairs = torch.empty(N, L, Hkv, 2, 16, 2, 2)
    if kind == "normal":
        pairs[..., 0] = 0.25 + 0.1 * torch.rand(N, L, Hkv, 2, 16, 2, generator=g)
        pairs[..., 1] = -7.5 * pairs[..., 0] + torch.randn(N, L, Hkv, 2, 16, 2, generator=g) * 0.5
    elif kind == "wide":  # scales over 2^20, some zero, minima of their own
        pairs[..., 0] = torch.pow(2.0, torch.randint(-16, 5, (N, L, Hkv, 2, 16, 2), generator=g).float())
        pairs[..., 0][torch.rand(N, L, Hkv, 2, 16, 2, generator=g) < 0.1] = 0
        pairs[..., 0, :, :, 0] *= 0.1
        pairs[..., 1] = torch.randn(N, L, Hkv, 2, 16, 2, generator=g)
    elif kind == "tiny":
        pairs[..., 0] = torch.rand(N, L, Hkv, 2, 16, 2, generator=g) * 2e-6
        pairs[..., 1] = torch.randn(N, L, Hkv, 2, 16, 2, generator=g) * 1e-5
    elif kind == "large":
        pairs[..., 0] = torch.rand(N, L, Hkv, 2, 16, 2, generator=g) * 4000
        pairs[..., 0, :, :, 0] *= 1e-4
        pairs[..., 1] = -7.5 * pairs[..., 0]
    cache[..., 1024:] = pairs.flatten(3).to(dtype)
    return cache


def _run(dev, q, cache, layer, tables, lens, scale=SCALE, **kw):
    out = torch.full_like(q, 7.0).to(dev)
    ops.paged_attention_decode_int4(out, q.to(dev), cache.to(dev) if cache.device.type == "cpu" else cache, layer,
                                    torch.as_tensor(tables).to(dev), torch.as_tensor(lens, dtype=torch.int32).to(dev), scale, **kw)
    return out.cpu()


def _check(dev, q, cache, layer, tables, lens, scale=SCALE, **kw):
    ops.read_device_errors(dev)
    got = _run(dev, q, cache, layer, tables, lens, scale, **kw)
    assert ops.read_device_errors(dev) == 0
    want = ref.attention(q, cache, layer, tables, lens, scale)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    bound = _bound(want, q, cache, layer, tables, lens, scale)
    assert (off <= bound).all(), f"off by {(off / bound).max():.3f} of the bound, {off.max():.3g}"
    return got


def _q(dtype, B, Hq, seed=1):
    return torch.randn(B, Hq, 128, generator=torch.Generator().manual_seed(seed)).to(dtype)


@BOTH
@pytest.mark.parametrize("lens", [[1], [16], [0, 1, 15, 16, 17, 31, 32, 33], [300, 5, 0, 129, 77]])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (4, 7), (2, 8), (1, 16), (3, 9), (8, 1)])
def test_lengths_and_groups(cuda_device, dtype, lens, Hkv, G):
    N = sum((n + 15) // 16 for n in lens) + 3
    _check(cuda_device, _q(dtype, len(lens), Hkv * G), _cache(dtype, N, 2, Hkv, 5), 1, make_tables(lens, N, 3), lens)


@BOTH
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 10, 11, 12, 13, 14, 15])
def test_every_group_size(cuda_device, dtype, G):
    lens = [40, 3, 200]
    _check(cuda_device, _q(dtype, 3, 2 * G, G), _cache(dtype, 24, 1, 2, G), 0, make_tables(lens, 24, G), lens)


@BOTH
@pytest.mark.parametrize("kind", ["wide", "tiny", "large"])
def test_scales_of_every_size(cuda_device, dtype, kind):
    lens = [500, 33, 1, 90]
    _check(cuda_device, _q(dtype, 4, 8), _cache(dtype, 60, 1, 2, 8, kind), 0, make_tables(lens, 60, 1), lens)


@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e8, 1e30])
def test_bf16_values_far_from_one(cuda_device, size):
    """Value scales of every size bf16 has, over 2^10 within a sequence."""
    dtype, lens = torch.bfloat16, [300, 20, 7]
    cache = _cache(dtype, 30, 1, 2, 8)
    g = torch.Generator().manual_seed(int(-math.log10(size)) % 97)
    s = size * torch.pow(2.0, -10 * torch.rand(30, 1, 2, 16, 2, generator=g))
    pairs = cache[..., 1088:].view(30, 1, 2, 16, 2, 2)
    pairs[..., 0] = s.to(dtype)
    pairs[..., 1] = (-7 * s + size * 0.1 * torch.randn(s.shape, generator=g)).to(dtype)
    q, tables = _q(dtype, 3, 8), make_tables(lens, 30, 1)
    got = _run(cuda_device, q, cache, 0, tables, lens)
    want = ref.attention(q, cache, 0, tables, lens, SCALE)
    assert ((got.double() - want).abs() <= _bound(want, q, cache, 0, tables, lens, SCALE)).all()


@BOTH
def test_long_sequences_split_over_many_warps(cuda_device, dtype):
    lens = [20000, 7, 9001]
    N = 2000
    _check(cuda_device, _q(dtype, 3, 8), _cache(dtype, N, 1, 1, 2), 0, make_tables(lens, N, 2), lens)


def test_many_tiles_in_one_warp_do_not_drift(cuda_device):
    """More pairs than worker warps: each warp sums hundreds of tiles, all of one sign."""
    dtype, B, Hkv = torch.float16, 3, 640
    lens = [2500, 2300, 2017]
    cache = _cache(dtype, 160, 1, Hkv, 4)
    tables = make_tables(lens, 500, 4) % 160  # blocks shared between sequences
    _check(cuda_device, _q(dtype, B, Hkv), cache, 0, tables, lens)


@BOTH
def test_an_outlier_token_leaves_the_others_their_precision(cuda_device, dtype):
    """One token's values are 4000 times the others', and no query looks at it."""
    cache = _cache(dtype, 8, 1, 1, 6)
    pairs = cache[..., 1024:].view(8, 1, 1, 2, 16, 2, 2)
    pairs[3, 0, 0, 1, 5, :, 0] = 1000.0
    pairs[3, 0, 0, 1, 5, :, 1] = -7500.0
    pairs[3, 0, 0, 0, 5, :, 0] = 0.0
    pairs[3, 0, 0, 0, 5, :, 1] = -8.0
    q = (_q(dtype, 1, 4).abs() + 0.5).to(dtype)
    tables = torch.arange(8, dtype=torch.int32).view(1, 8).numpy()
    got = _run(cuda_device, q, cache, 0, tables, [128])
    want = ref.attention(q, cache, 0, tables, [128], SCALE)
    seen = cache.clone()
    seen[3, 0, 0, 1088:].view(16, 2, 2)[5] = 0
    off = (got.double() - want).abs()
    # its weight is below 2^-30, so that the bound of the values without it holds
    assert (off <= _bound(want, q, seen, 0, tables, [128], SCALE) + 1e-5).all()


@BOTH
def test_what_lies_past_the_end_does_not_count(cuda_device, dtype):
    """NaN, infinities and the largest values in unused rows, unused blocks and padding of the table."""
    lens = [5, 33, 16]
    cache = _cache(dtype, 12, 1, 2, 9)
    tables = make_tables(lens, 10, 2, width=6)
    dirty = cache.clone()
    used = {int(b) for row, n in zip(tables, lens) for b in row[:(n + 15) // 16]}
    for b in range(12):
        if b not in used:
            dirty[b] = float("nan")
    fill = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max])
    for row, n in zip(tables, lens):
        if n % 16:
            pairs = dirty[int(row[n // 16]), 0, :, 1024:].view(2, 2, 16, 2, 2)
            pairs[:, :, n % 16:] = fill[torch.arange(pairs[:, :, n % 16:].numel()) % 4].view_as(pairs[:, :, n % 16:]).to(dtype)
    tables[0, 1:], tables[2, 1:] = 11, 10
    q = _q(dtype, 3, 8)
    clean = _check(cuda_device, q, cache, 0, tables, lens)
    assert torch.equal(_run(cuda_device, q, dirty, 0, tables, lens), clean)


@BOTH
def test_a_poisoned_row_shows(cuda_device, dtype):
    cache = _cache(dtype, 6, 1, 2, 1)
    key = torch.randn(1, 2, 128).to(dtype)
    value = key.clone()
    value[0, 1, 3] = float("nan")
    ref.write(cache, 0, key, value, [2 * 16 + 4])
    tables = torch.arange(6, dtype=torch.int32).view(1, 6).numpy()
    got = _run(cuda_device, _q(dtype, 1, 4), cache, 0, tables, [90])
    bad = torch.zeros(4, 128, dtype=torch.bool)
    bad[2:, :64] = True
    assert torch.equal(torch.isnan(got[0]), bad)


@BOTH
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.5, 1e-30])
def test_scales_of_the_scores(cuda_device, dtype, scale):
    lens = [70, 1, 400]
    _check(cuda_device, _q(dtype, 3, 6), _cache(dtype, 36, 1, 3, 3), 0, make_tables(lens, 36, 1), lens, scale)


@BOTH
@pytest.mark.parametrize("off", [0, 1, 2, 8])
def test_strided_query_and_output(cuda_device, dtype, off):
    B, Hq, lens = 3, 4, [33, 2, 64]
    cache, tables = _cache(dtype, 9, 1, 2, 3), make_tables(lens, 9, 1)
    fused = torch.randn(B, 6 * 128 + 16, generator=torch.Generator().manual_seed(off)).to(dtype)
    q_off = off - off % 2  # the query is 4-byte aligned
    dev = fused.to(cuda_device)
    q = dev[:, q_off:q_off + Hq * 128].view(B, Hq, 128)
    wide = torch.full((B, 6 * 128 + 16), 3.0, dtype=dtype, device=cuda_device)
    out = wide[:, off:off + Hq * 128].view(B, Hq, 128)
    args = (cache.to(cuda_device), 0, torch.as_tensor(tables).to(cuda_device), torch.tensor(lens, dtype=torch.int32, device=cuda_device), SCALE)
    ops.paged_attention_decode_int4(out, q, *args)
    host_q = fused[:, q_off:q_off + Hq * 128].reshape(B, Hq, 128)
    want = ref.attention(host_q, cache, 0, tables, lens, SCALE)
    assert ((out.cpu().double() - want).abs() <= _bound(want, host_q, cache, 0, tables, lens, SCALE)).all()
    assert (wide[:, :off] == 3).all() and (wide[:, off + Hq * 128:] == 3).all()


def test_same_result_as_the_16bit_kernel_on_the_values(cuda_device):
    """The two kernels on the same values, read back into a 16-bit cache. 16-bit values differ from the
    4-bit cache's by their own rounding, of which the weighted mean keeps at most the largest."""
    dtype, lens, N, Hkv = torch.bfloat16, [200, 16, 1, 999], 90, 4
    cache, tables = _cache(dtype, N, 1, Hkv, 12).to(cuda_device), torch.as_tensor(make_tables(lens, N, 5)).to(cuda_device)
    k, v = ops.gather_cache_int4(cache, 0, torch.arange(16 * N, device=cuda_device))
    kv = torch.stack([k.view(N, 16, Hkv, 128), v.view(N, 16, Hkv, 128)], 1).unsqueeze(1).contiguous()
    q, sl = _q(dtype, 4, 32).to(cuda_device), torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.paged_attention_decode_int4(a, q, cache, 0, tables, sl, SCALE)
    ops.paged_attention_decode(b, q, kv, 0, tables, sl, SCALE)
    assert (a.float() - b.float()).norm() <= 4 * 2.0 ** -8 * b.float().norm()


def test_repeats_prefetch_and_plan_reuse_give_the_same_bits(cuda_device):
    dtype, lens, N = torch.float16, [3000, 40, 0, 177, 16], 250
    cache, tables = _cache(dtype, N, 3, 2, 12).to(cuda_device), torch.as_tensor(make_tables(lens, N, 5)).to(cuda_device)
    sl, q = torch.tensor(lens, dtype=torch.int32, device=cuda_device), _q(dtype, 5, 14).to(cuda_device)
    plan = ops.DecodePlan(5, 14, 2, 128, cuda_device, cache="int4").plan(sl, tables)
    first = None
    for prefetch in (False, True, True):
        outs = [torch.empty_like(q) for _ in range(3)]
        for layer in range(3):
            ops.paged_attention_decode_int4(outs[layer], q, cache, layer, tables, sl, SCALE, plan=plan, prefetch=prefetch)
        first = first or outs
        assert all(torch.equal(a, b) for a, b in zip(first, outs))
    assert not first[0][2].any()
    assert ops.read_device_errors(cuda_device) == 0


def test_ids_and_lengths_outside_are_left_out_and_reported(cuda_device):
    dtype, lens = torch.bfloat16, [40, 100, 33]
    cache, tables = _cache(dtype, 14, 1, 2, 7), make_tables(lens, 14, 3)
    q = _q(dtype, 3, 4)
    clean = _run(cuda_device, q, cache, 0, tables, lens)
    for bad in (14, -1, 1 << 30):
        t = tables.copy()
        t[0, 1] = bad
        ops.read_device_errors(cuda_device)
        got = _run(cuda_device, q, cache, 0, t, lens)
        assert ops.read_device_errors(cuda_device) == AEG_DEVERR_BLOCK_ID_RANGE
        assert torch.equal(got[1:], clean[1:])
        # the block's tokens are left out: as if only blocks 0 and 2 were there
        short = torch.as_tensor(tables)[:1, [0, 2]].numpy()
        want = ref.attention(q[:1], cache, 0, short, [24], SCALE)
        assert ((got[:1].double() - want).abs() <= _bound(want, q[:1], cache, 0, short, [24], SCALE)).all()
    got = _run(cuda_device, q, cache, 0, tables, [40, 16 * tables.shape[1] + 5, -3])
    assert ops.read_device_errors(cuda_device) == AEG_DEVERR_SEQ_LEN_RANGE
    assert torch.equal(got[0], clean[0]) and not got[2].any()


def test_a_plan_of_the_other_kind_is_refused(cuda_device):
    lens = [40, 3]
    cache, tables = _cache(torch.float16, 6, 1, 2, 7).to(cuda_device), torch.as_tensor(make_tables(lens, 6, 3)).to(cuda_device)
    sl, q = torch.tensor(lens, dtype=torch.int32, device=cuda_device), _q(torch.float16, 2, 4).to(cuda_device)
    out = torch.empty_like(q)
    wrong = ops.DecodePlan(2, 4, 2, 128, cuda_device).plan(sl, tables)
    with pytest.raises(ValueError, match="plan"):
        ops.paged_attention_decode_int4(out, q, cache, 0, tables, sl, SCALE, plan=wrong)
    kv = torch.zeros(6, 1, 2, 16, 2, 128, dtype=torch.float16, device=cuda_device)
    right = ops.DecodePlan(2, 4, 2, 128, cuda_device, cache="int4").plan(sl, tables)
    with pytest.raises(ValueError, match="plan"):
        ops.paged_attention_decode(out, q, kv, 0, tables, sl, SCALE, plan=right)
    ops.read_device_errors(cuda_device)
    wrong.cache = "int4"  # past the host's check the kernel notices the plan's number of workers
    ops.paged_attention_decode_int4(out, q, cache, 0, tables, sl, SCALE, plan=wrong)
    assert ops.read_device_errors(cuda_device) & AEG_DEVERR_PLAN_MISMATCH


def test_refusals_and_empty_batch(cuda_device):
    lens = [40, 3]
    cache, tables = _cache(torch.float16, 6, 1, 2, 7).to(cuda_device), torch.as_tensor(make_tables(lens, 6, 3)).to(cuda_device)
    sl, q = torch.tensor(lens, dtype=torch.int32, device=cuda_device), _q(torch.float16, 2, 4).to(cuda_device)
    good = dict(out=torch.empty_like(q), query=q, kv_cache=cache, layer=0, block_tables=tables, seq_lens=sl, scale=SCALE)
    ops.paged_attention_decode_int4(**good)
    for bad in (dict(query=q.bfloat16()), dict(query=q[:, :3], out=good["out"][:, :3]), dict(kv_cache=cache.bfloat16()), dict(layer=1),
                dict(layer=-1), dict(seq_lens=sl.long()), dict(block_tables=tables[:1]), dict(out=good["out"][:, :2]), dict(out=q.float()),
                dict(block_tables=tables[:, :0]), dict(scale=float("nan")), dict(scale=float("inf")), dict(kv_cache=cache[:, :, :, :1151]), dict(query=q.cpu()), dict(seq_lens=sl.cpu()),
                dict(query=torch.empty(2, 34, 128, dtype=torch.float16, device=cuda_device), out=torch.empty(2, 34, 128, dtype=torch.float16, device=cuda_device))):
        with pytest.raises((ValueError, NotImplementedError)):
            ops.paged_attention_decode_int4(**dict(good, **bad))
    with pytest.raises(ValueError, match="cache"):
        ops.DecodePlan(2, 4, 2, 128, cuda_device, cache="fp8")
    none = q[:0]
    ops.paged_attention_decode_int4(none, none, cache, 0, tables[:0], sl[:0], SCALE)


def test_two_streams_with_plans_of_their_own(cuda_device):
    dtype, lens, N = torch.bfloat16, [3000, 500, 1200], 300
    cache, tables = _cache(dtype, N, 1, 4, 12).to(cuda_device), torch.as_tensor(make_tables(lens, N, 5)).to(cuda_device)
    sl, q = torch.tensor(lens, dtype=torch.int32, device=cuda_device), _q(dtype, 3, 16).to(cuda_device)
    alone = torch.empty_like(q)
    ops.paged_attention_decode_int4(alone, q, cache, 0, tables, sl, SCALE)
    kv = torch.randn(N, 1, 2, 16, 4, 128, device=cuda_device).to(dtype)
    alone16 = torch.empty_like(q)
    ops.paged_attention_decode(alone16, q, kv, 0, tables, sl, SCALE)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            plan = ops.DecodePlan(3, 16, 4, 128, cuda_device, cache="int4").plan(sl, tables)
            plan16 = ops.DecodePlan(3, 16, 4, 128, cuda_device).plan(sl, tables)
            for _ in range(5):
                outs.append((torch.empty_like(q), torch.empty_like(q), plan, plan16))
                ops.paged_attention_decode_int4(outs[-1][0], q, cache, 0, tables, sl, SCALE, plan=plan, prefetch=True)
                ops.paged_attention_decode(outs[-1][1], q, kv, 0, tables, sl, SCALE, plan=plan16, prefetch=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, alone) and torch.equal(b, alone16) for a, b, *_ in outs)
    assert ops.read_device_errors(cuda_device) == 0


def test_captured_step_replays_on_new_lengths(cuda_device):
    dtype, N = torch.float16, 40
    cache = _cache(dtype, N, 2, 2, 3)
    tables = make_tables([160, 160, 160], N, 3)
    dev_tables, dev_cache = torch.as_tensor(tables).to(cuda_device), cache.to(cuda_device)
    sl, q = torch.tensor([30, 1, 160], dtype=torch.int32, device=cuda_device), _q(dtype, 3, 8).to(cuda_device)
    plan = ops.DecodePlan(3, 8, 2, 128, cuda_device, cache="int4")
    outs = [torch.empty_like(q) for _ in range(2)]

    def step():
        plan.plan(sl, dev_tables)
        for layer in range(2):
            ops.paged_attention_decode_int4(outs[layer], q, dev_cache, layer, dev_tables, sl, SCALE, plan=plan, prefetch=layer > 0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([30, 1, 160], [0, 77, 16], [159, 160, 144]):
        sl.copy_(torch.tensor(lens))
        q.copy_(_q(dtype, 3, 8, sum(lens)))
        graph.replay()
        for layer in range(2):
            want = ref.attention(q.cpu(), cache, layer, tables, lens, SCALE)
            assert ((outs[layer].cpu().double() - want).abs() <= _bound(want, q.cpu(), cache, layer, tables, lens, SCALE)).all()


def test_offsets_beyond_32_bits(cuda_device):
    """Blocks at the far end of a cache of 5.2 GB: written, read back and attended to."""
    dtype, L, Hkv, N = torch.bfloat16, 56, 40, 1000
    cache = torch.zeros(N, *layout.int4_block_shape(L, Hkv), dtype=dtype, device=cuda_device)
    g = torch.Generator().manual_seed(3)
    key, value = (torch.randn(20, Hkv, 128, generator=g).to(dtype) for _ in range(2))
    blocks = [998, 999]
    slots = torch.tensor([blocks[i // 16] * 16 + i % 16 for i in range(20)])
    ops.reshape_and_cache_int4(key.to(cuda_device), value.to(cuda_device), cache, 55, slots.to(cuda_device))
    small = torch.zeros(2, *layout.int4_block_shape(1, Hkv), dtype=dtype)
    ref.write(small, 0, key, value, range(20))
    assert torch.equal(cache[998:, 55].cpu().view(torch.int16), small[:, 0].view(torch.int16))
    assert not cache[:998].view(torch.int32).any() and not cache[998:, :55].view(torch.int32).any()
    k, _ = ops.gather_cache_int4(cache, 55, slots.to(cuda_device))
    assert torch.equal(k.cpu().view(torch.int16), ref.gather(small, 0, range(20))[0].view(torch.int16))
    q = _q(dtype, 1, Hkv)
    got = _run(cuda_device, q, cache, 55, torch.tensor([blocks], dtype=torch.int32), [20])
    want = ref.attention(q, small, 0, [[0, 1]], [20], SCALE)
    assert ((got.double() - want).abs() <= _bound(want, q, small, 0, [[0, 1]], [20], SCALE)).all()
