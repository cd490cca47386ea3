"""The oracle of the 4-bit cache, the rotary positions and the shared blocks against exact
arithmetic and its own inverses, and what the calls refuse (no GPU needed)."""
import ctypes
import random

import numpy as np
import pytest
import torch

from aegaeon_b200 import _native, layout, ops
from oracle import serving_ref as ref

INVAL, UNSUP = _native.AEG_ERR_INVALID_ARGUMENT, _native.AEG_ERR_UNSUPPORTED


def _hard_rows(dtype, n, g):
    """Rows of 64 where rounding is easiest to get wrong: coarse grids full of ties, tiny spreads,
    large offsets, subnormals, widely different magnitudes, constants."""
    kinds = [torch.randint(-8, 9, (n, 64), generator=g) / 4.0,
             torch.randint(0, 31, (n, 64), generator=g) * 0.5 + 100,
             torch.randn(n, 64, generator=g) * 1e-6,
             torch.randn(n, 64, generator=g) * torch.pow(2.0, torch.randint(-20, 10, (n, 64), generator=g)),
             torch.randn(n, 64, generator=g) + 300,
             torch.full((n, 64), 3.25),
             torch.randn(n, 64, generator=g) * (6e4 if dtype == torch.float16 else 1e37)]
    return torch.cat([k.to(dtype) for k in kinds])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantise_matches_exact_fractions(dtype):
    rows = _hard_rows(dtype, 6, torch.Generator().manual_seed(3))
    rows = rows[torch.isfinite(rows).all(1)]
    codes, pairs = ref.quantise(torch.cat([rows, rows], 1))
    for i, row in enumerate(rows):
        c, s, lo = ref.quantise_fraction([float(v) for v in row], dtype)
        assert codes[i, :64].tolist() == c and codes[i, 64:].tolist() == c
        assert pairs[i].double().tolist() == [[s, lo], [s, lo]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tile_layout_holds_every_element_once(dtype):
    both = torch.cat([ref.KEY_AT.flatten(), ref.VALUE_AT.flatten()])
    places = 2 * both + (torch.arange(128).repeat(32) % 2)
    assert torch.equal(places.sort().values, torch.arange(4096))
    g = torch.Generator().manual_seed(0)
    cache = torch.zeros(3, *layout.int4_block_shape(2, 4), dtype=dtype)
    key, value = (torch.randn(40, 4, 128, generator=g).to(dtype) for _ in range(2))
    slots = torch.randperm(48, generator=g)[:40]
    ref.write(cache, 1, key, value, slots)
    k, v = ref.gather(cache, 1, slots)
    for x, y in ((key, k), (value, v)):
        codes, pairs = ref.quantise(x)
        want = codes.double().unflatten(-1, (2, 64)) * pairs[..., :1].double() + pairs[..., 1:].double()
        assert torch.equal(y, want.flatten(-2).float().to(dtype))
        # half a scale, its rounding (at code 15) and the read-back's rounding
        step = (x.double().unflatten(-1, (2, 64)).amax(-1) - x.double().unflatten(-1, (2, 64)).amin(-1)) / 15
        far = (y.double() - x.double()).abs().unflatten(-1, (2, 64)).amax(-1)
        assert (far <= step * (0.5 + 15.5 * ref.half_step(dtype)) + 8 * ref.half_step(dtype)).all()
    assert not cache[:, 0].view(torch.int16).any()


def test_int4_block_shape():
    assert layout.int4_block_shape(28, 4) == (28, 4, 1152)
    with pytest.raises(NotImplementedError):
        layout.int4_block_shape(2, 4, 64)


def test_interleaved_axes_deal_in_turn():
    assert list(ops._axis_of((3, 1, 2), True)) == [0, 1, 2, 0, 2, 0] == ref.axes_of((3, 1, 2), True)
    assert list(ops._axis_of((3, 1, 2), False)) == [0, 0, 0, 1, 2, 2]
    for bad in ((), (0, 0), (1, -1), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError, match="sections"):
            ops._axis_of(bad, False)


def test_pool_oracle_round_trip():
    r = random.Random(5)
    pool = ref.Pool([0] * 40, [[0] * 4 for _ in range(8)], [0] * 8, None)
    for row in range(3):
        pool.tables[row] = list(range(4 * row, 4 * row + 4))
        pool.lens[row] = [64, 33, 1][row]
        for b in pool.tables[row][:(pool.lens[row] + 15) // 16]:
            pool.counts[b] += 1
    start = list(pool.counts)
    new, errors = pool.fork([0, 1, 2, 1, 9], [3, 4, 5, 4, 6])
    assert errors == {"entry"} and new == [-1, 7, 9, -1, -1]
    assert not pool.free([3, 4, 5, 5]) and pool.counts == start
    tables, counts, remap, n = pool.compact()
    assert n == sum(c > 0 for c in start) and counts[n:] == [0] * (40 - n) and r.random() < 1
    assert sorted(x for x in remap if x >= 0) == list(range(n))


def _aligned():
    buf = np.zeros(1 << 14, np.int64)
    return (buf.ctypes.data + 255) // 256 * 256, buf


def test_int4_calls_refuse_on_the_host():
    p, _k = _aligned()
    lib = _native.lib
    good = dict(k=p, v=p, ks=512, vs=512, c=p, bs=4 * 1152, n=8, s=p, T=4, H=4, D=128, t=0)

    for fn in (lib.aeg_reshape_and_cache_int4, lib.aeg_gather_cache_int4):
        def call(**kw):
            a = dict(good, **kw)
            return fn(*([a["k"], a["v"], a["ks"], a["vs"], a["c"]] + [a["bs"], a["n"], a["s"], a["T"], a["H"], a["D"], a["t"], None]))

        assert call(T=0) == 0 and call(T=0, k=None, c=None) == 0
        assert call(T=-1) == INVAL and call(T=1 << 31) == INVAL
        assert call(H=0) == INVAL and call(D=0) == INVAL and call(D=64) == UNSUP and call(t=2) == INVAL
        assert call(k=None) == INVAL and call(c=None) == INVAL and call(s=None) == INVAL
        assert call(ks=511) == INVAL and call(vs=100) == INVAL
        assert call(bs=4 * 1152 - 8) == INVAL and call(bs=4 * 1152 + 4) == INVAL
        assert call(c=p + 8) == INVAL and call(k=p + 1) == INVAL and call(s=p + 4) == INVAL
        assert call(n=-1) == INVAL


def test_int4_attention_refuses_on_the_host():
    p, _k = _aligned()
    lib = _native.lib
    need = lib.aeg_decode_workspace_size(2, 8, 2, 128)
    assert lib.aeg_decode_plan_int4(p, need, p, 4, p, 2, 8, 2, 64, None) == UNSUP
    assert lib.aeg_decode_plan_int4(p, need, p, 4, p, 2, 34, 2, 128, None) == INVAL
    assert lib.aeg_decode_plan_int4(p + 8, need, p, 4, p, 2, 8, 2, 128, None) == INVAL
    assert lib.aeg_decode_plan_int4(p, need - 1, p, 4, p, 2, 8, 2, 128, None) == INVAL
    assert lib.aeg_decode_plan_int4(p, need, None, 4, p, 2, 8, 2, 128, None) == INVAL
    good = dict(o=p, os=1024, q=p, qs=1024, c=p, bs=2 * 1152, n=8, t=p, W=4, sl=p, B=2, Hq=8, Hkv=2, D=128, dt=0, ws=p, wsb=need, f=0)

    def call(**kw):
        a = dict(good, **kw)
        return lib.aeg_paged_attn_decode_int4(a["o"], a["os"], a["q"], a["qs"], a["c"], a["bs"], a["n"], a["t"], a["W"], a["sl"],
                                              a["B"], a["Hq"], a["Hkv"], a["D"], 0.1, a["dt"], a["ws"], a["wsb"], a["f"], None)

    assert call(B=0) == 0 and call(B=-1) == INVAL
    assert call(D=64) == UNSUP and call(Hq=9) == INVAL and call(Hq=34) == INVAL and call(dt=3) == INVAL and call(W=0) == INVAL
    assert call(o=None) == INVAL and call(q=None) == INVAL and call(c=None) == INVAL and call(t=None) == INVAL and call(sl=None) == INVAL
    assert call(os=1000) == INVAL and call(qs=1000) == INVAL and call(qs=1025) == INVAL and call(q=p + 2) == INVAL and call(o=p + 1) == INVAL
    assert call(bs=2 * 1152 - 8) == INVAL and call(bs=2 * 1152 + 4) == INVAL and call(c=p + 8) == INVAL
    assert call(n=0) == INVAL and call(n=1 << 31) == INVAL
    assert call(ws=None) == INVAL and call(ws=p + 16) == INVAL and call(wsb=need - 1) == INVAL
    assert call(f=2) == INVAL and call(f=4) == INVAL


def test_rotary_refuses_on_the_host():
    p, _k = _aligned()
    lib = _native.lib
    good = dict(qo=p, qos=1024, ko=p, kos=256, q=p, qs=1024, k=p, ks=256, pos=p, ps=4, axes=3, inv=p,
                ax=bytes([0] * 32 + [1] * 16 + [2] * 16), half=64, T=4, Hq=8, Hkv=2, D=128, t=0)

    def call(**kw):
        a = dict(good, **kw)
        return lib.aeg_rotary_multi_axis(a["qo"], a["qos"], a["ko"], a["kos"], a["q"], a["qs"], a["k"], a["ks"], a["pos"],
                                         a["ps"], a["axes"], a["inv"], a["ax"], a["half"], 1.0, a["T"], a["Hq"],
                                         a["Hkv"], a["D"], a["t"], None)

    assert call(T=0) == 0
    assert call(T=-1) == INVAL and call(Hq=0) == INVAL and call(Hkv=-1) == INVAL and call(D=0) == INVAL and call(t=5) == INVAL
    assert call(axes=0) == INVAL and call(axes=5) == INVAL and call(half=0) == INVAL and call(half=65) == INVAL
    assert call(axes=2) == INVAL and "names axis 2" in _native.last_error()
    assert call(D=512, half=129, Hq=1, Hkv=0, ax=bytes(129)) == UNSUP
    assert call(q=None) == INVAL and call(k=None) == INVAL and call(pos=None) == INVAL and call(inv=None) == INVAL
    assert call(ax=None) == INVAL
    assert call(qs=1000) == INVAL and call(qos=1000) == INVAL and call(ks=255) == INVAL and call(kos=255) == INVAL
    assert call(ps=-1) == INVAL and call(q=p + 1) == INVAL and call(pos=p + 4) == INVAL


def test_shared_block_calls_refuse_on_the_host():
    p, _k = _aligned()
    lib = _native.lib
    assert lib.aeg_fork_blocks_workspace_size(0) == 0 and lib.aeg_fork_blocks_workspace_size(10) >= 10 * 24
    assert lib.aeg_compact_blocks_workspace_size(100) >= 416 and lib.aeg_compact_blocks_workspace_size(-1) == 0
    good = dict(pool=p, bb=64, N=8, rc=p, tb=p, W=4, R=4, sl=p, src=p, dst=p, n=2, new=p, ws=p, wsb=1 << 14)

    def fork(**kw):
        a = dict(good, **kw)
        return lib.aeg_fork_blocks(a["pool"], a["bb"], a["N"], a["rc"], a["tb"], a["W"], a["R"], a["sl"], a["src"],
                                   a["dst"], a["n"], a["new"], a["ws"], a["wsb"], None)

    assert fork(n=0) == 0 and fork(n=-1) == INVAL and fork(n=1 << 25) == INVAL
    assert fork(N=-1) == INVAL and fork(N=1 << 31) == INVAL and fork(W=0) == INVAL and fork(R=-1) == INVAL
    assert fork(rc=None) == INVAL and fork(tb=None) == INVAL and fork(sl=None) == INVAL and fork(pool=None) == INVAL
    assert fork(src=None) == INVAL and fork(dst=None) == INVAL and fork(new=None) == INVAL
    assert fork(src=p + 4) == INVAL and fork(rc=p + 2) == INVAL
    assert fork(ws=None) == INVAL and fork(ws=p + 8) == INVAL and fork(wsb=8) == INVAL

    def free(**kw):
        a = dict(good, **kw)
        return lib.aeg_free_blocks(a["N"], a["rc"], a["tb"], a["W"], a["R"], a["sl"], a["src"], a["n"], None)

    assert free(n=0) == 0 and free(n=-1) == INVAL and free(src=None) == INVAL and free(src=p + 4) == INVAL
    assert free(rc=None) == INVAL and free(W=0) == INVAL

    def compact(**kw):
        a = dict(dict(good, rco=p + 64, tbo=p, remap=p, live=p), **kw)
        return lib.aeg_compact_blocks(a["pool"], a["bb"], a["N"], a["rc"], a["tb"], a["W"], a["R"], a["sl"], a["rco"],
                                      a["tbo"], a["remap"], a["live"], a["ws"], a["wsb"], None)

    assert compact(N=-1) == INVAL and compact(pool=None) == INVAL and compact(rco=None) == INVAL
    assert compact(rco=p) == INVAL and compact(remap=None) == INVAL and compact(live=None) == INVAL
    assert compact(tbo=None) == INVAL and compact(ws=None) == INVAL and compact(wsb=15) == INVAL
    assert compact(remap=p + 2) == INVAL


def test_wrappers_refuse_host_tensors():
    kv = torch.zeros(4, 1, 4, 1152, dtype=torch.float16)
    row = torch.zeros(2, 4, 128, dtype=torch.float16)
    ids = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.reshape_and_cache_int4(row, row, kv, 0, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.reshape_and_cache_int4(None, None, kv, 0, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.gather_cache_int4(kv, 0, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary_multi_axis(row, row, torch.zeros(3, 2, dtype=torch.int64), torch.zeros(64), [64, 0, 0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.fork_blocks(kv, ids, ids.view(2, 2), ids[:2], [0], [1])
    with pytest.raises(ValueError, match="CUDA"):
        ops.free_blocks(ids, ids.view(2, 2), ids[:2], [0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.compact_blocks(kv, ids, ids.view(2, 2), ids[:2])
    assert ctypes.sizeof(ctypes.c_void_p) == 8
