"""Rotary positions with several axes against the formula in 64 bits.

Tolerance: the output's own rounding (half a step of its value, or of the least subnormal) and the
fp32 work before it, relative to |a| + |b|: 2^-22 for the reduced turn's rounding and the sine and
cosine (each within 2^-22), 2^-22 for the products and sums."""
import pytest
import torch

from aegaeon_b200 import ops
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu


def _check(out, x, positions, inv, sections, interleaved, scaling=1.0):
    half = inv.numel()
    want = ref.rotary(x, positions, inv, sections, interleaved, scaling)
    a, b = x[..., :half].double().abs(), x[..., half:2 * half].double().abs()
    near = torch.cat([a + b, a + b, torch.zeros_like(x[..., 2 * half:].double())], -1) * scaling
    info = torch.finfo(x.dtype)
    bound = want.abs() * info.eps / 2 + near * 2.0 ** -20 + info.smallest_normal * info.eps / 2
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,Hq,Hkv,D,sections", [
    (1, 1, 1, 128, (16, 24, 24)), (1, 28, 4, 128, (64,)), (5, 8, 2, 64, (8, 12, 12)), (33, 7, 1, 80, (10, 15, 15)),
    (64, 32, 4, 128, (24, 20, 20)), (17, 3, 3, 96, (5, 6, 7)), (9, 40, 40, 128, (0, 64, 0)), (3000, 4, 2, 128, (16, 24, 24)),
    (11, 2, 2, 256, (40, 40, 48)), (4, 5, 1, 130, (1, 1)), (2, 3, 1, 7, (1, 1, 1)), (6, 64, 8, 128, (16, 16, 16, 16))])
@pytest.mark.parametrize("interleaved", [False, True])
def test_matches_the_formula(cuda_device, dtype, T, Hq, Hkv, D, sections, interleaved):
    g = torch.Generator().manual_seed(T + D)
    q, k = (torch.randn(T, h, D, generator=g).to(dtype) for h in (Hq, Hkv))
    pos = torch.randint(0, 200000, (len(sections), T), generator=g)
    half = sum(sections)
    inv = (1.0 / 1e6 ** (torch.arange(half) / half)).float()
    qo, ko = ops.rotary_multi_axis(q.to(cuda_device), k.to(cuda_device), pos.to(cuda_device), inv.to(cuda_device), sections,
                                   interleaved=interleaved)
    _check(qo.cpu(), q, pos, inv, sections, interleaved)
    _check(ko.cpu(), k, pos, inv, sections, interleaved)


@pytest.mark.parametrize("first", [0, (1 << 20) - 3, -5, (1 << 31) - 2])
def test_far_and_negative_positions(cuda_device, first):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(6, 2, 128, generator=g).to(torch.float16) for _ in range(2))
    pos = first + torch.arange(6)
    inv = (1.0 / 1e4 ** (torch.arange(64) / 64)).float()
    qo, ko = ops.rotary_multi_axis(q.to(cuda_device), k.to(cuda_device), pos.to(cuda_device), inv.to(cuda_device), (64,),
                                   scaling=1.25)
    _check(qo.cpu(), q, pos.view(1, -1), inv, (64,), False, 1.25)
    _check(ko.cpu(), k, pos.view(1, -1), inv, (64,), False, 1.25)


@pytest.mark.parametrize("off", [0, 1, 2, 8])
def test_in_place_on_views_of_a_fused_projection(cuda_device, off):
    T, Hq, Hkv = 19, 4, 2
    qkv = torch.randn(T, (Hq + 2 * Hkv) * 128 + 8, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    dev = qkv.to(cuda_device)
    pos = torch.stack([torch.arange(T), torch.arange(T) // 4, torch.arange(T) % 4]) + 900
    inv = (1.0 / 1e4 ** (torch.arange(48) / 48)).float()

    def views(t):
        return (t[:, off:off + Hq * 128].view(T, Hq, 128), t[:, off + Hq * 128:off + (Hq + Hkv) * 128].view(T, Hkv, 128))

    q, k = views(dev)
    ops.rotary_multi_axis(q, k, pos.to(cuda_device), inv.to(cuda_device), (16, 16, 16), query_out=q, key_out=k)
    for x, y in zip(views(dev.cpu()), views(qkv)):
        _check(x, y, pos, inv, (16, 16, 16), False)
    assert torch.equal(dev[:, off + (Hq + Hkv) * 128:].cpu(), qkv[:, off + (Hq + Hkv) * 128:])
    assert torch.equal(dev[:, :off].cpu(), qkv[:, :off])


def test_sliced_positions_empty_call_and_refusals(cuda_device):
    x = torch.randn(3, 2, 128, device=cuda_device).half()
    inv = torch.full((64,), 0.5, device=cuda_device)
    wide = torch.randint(0, 99, (3, 10), device=cuda_device)
    got = ops.rotary_multi_axis(x, x, wide[:, 2:5], inv, (16, 24, 24))[0]
    assert torch.equal(got, ops.rotary_multi_axis(x, x, wide[:, 2:5].contiguous(), inv, (16, 24, 24))[0])
    got = ops.rotary_multi_axis(x, x, wide.T[2:5].T, inv, (16, 24, 24))[0]
    assert torch.equal(got, ops.rotary_multi_axis(x, x, wide[:, 2:5], inv, (16, 24, 24))[0])
    one = wide[0, 2:5]
    got = ops.rotary_multi_axis(x, x, one.expand(3, -1), inv, (16, 24, 24))[0]
    assert torch.equal(got, ops.rotary_multi_axis(x, x, one, inv, (64,))[0])
    got = ops.rotary_multi_axis(x[:0], x[:0], wide[:, :0], inv, (16, 24, 24))
    assert got[0].shape == (0, 2, 128)
    pos = wide[:, :3]
    for a in (dict(sections=(16, 24)), dict(sections=(16, 24, 23)), dict(pos=pos.int()), dict(inv=inv.double()),
              dict(k=x.bfloat16()), dict(k=x[:2]), dict(k=x[..., :64]), dict(pos=pos[:, :2]), dict(q=x.float(), k=x.float()),
              dict(sections=(100, 100, 100), inv=torch.ones(300, device=cuda_device))):
        a = dict(dict(q=x, k=x, pos=pos, inv=inv, sections=(16, 24, 24)), **a)
        with pytest.raises((ValueError, NotImplementedError)):
            ops.rotary_multi_axis(a["q"], a["k"], a["pos"], a["inv"], a["sections"])
    with pytest.raises(ValueError, match="query_out"):
        ops.rotary_multi_axis(x, x, pos, inv, (16, 24, 24), query_out=x.float())


def test_on_another_stream_behind_the_producer(cuda_device):
    side = torch.cuda.Stream()
    x = torch.empty(2000, 8, 128, dtype=torch.bfloat16, device=cuda_device)
    pos = torch.arange(2000, device=cuda_device)
    inv = torch.rand(64, device=cuda_device)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x.copy_(torch.randn(2000, 8, 128))
        q, _ = ops.rotary_multi_axis(x, x, pos, inv, (64,))
    side.synchronize()
    _check(q.cpu(), x.cpu(), pos.cpu().view(1, -1), inv.cpu(), (64,), False)
