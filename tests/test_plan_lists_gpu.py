"""The two ways a plan's lists are written: over the GPU from the scans, and by the plan's one CTA where the
pairs' records do not fit the partial-result area (B * Hkv above about 133,000 times the group size with a
workspace, 38,000 with the allocation-free call's scratch)."""
import ctypes
import math

import pytest
import torch

from aegaeon_b200 import layout, ops
from aegaeon_b200._native import AEG_DTYPE_FP16, check, lib

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(128)


def _case(dev, B, Hkv, longest, seed):
    g = torch.Generator(dev).manual_seed(seed)
    W = (longest + 15) // 16
    lens = torch.randint(0, longest + 1, (B,), generator=g, device=dev).to(torch.int32)
    kv = torch.randn(9, *layout.kv_block_shape(1, Hkv, 128), generator=g, device=dev).half()  # shared by all sequences
    tables = torch.randint(0, 9, (B, W), generator=g, device=dev).to(torch.int32)
    q = torch.randn(B, Hkv, 128, generator=g, device=dev).half()
    return lens, kv, tables, q


def _reference(lens, kv, tables, q):
    """fp32, a few sequences at a time."""
    out = torch.zeros_like(q, dtype=torch.float32)
    for b0 in range(0, q.size(0), 64):
        rows = kv[tables[b0:b0 + 64].long(), 0]  # sequences, blocks, key/value, 16, heads, 128
        k, v = (rows[:, :, i].flatten(1, 2).float() for i in (0, 1))
        n = lens[b0:b0 + 64]
        seen = (torch.arange(k.size(1), device=q.device) < n.view(-1, 1)).unsqueeze(1)
        s = torch.einsum("bhd,bthd->bht", q[b0:b0 + 64].float(), k) * SCALE
        p = torch.where(seen, torch.exp(s - torch.where(seen, s, -math.inf).amax(-1, keepdim=True)), 0.0).nan_to_num()
        o = torch.einsum("bht,bthd->bhd", p, v) / p.sum(-1, keepdim=True)
        out[b0:b0 + 64] = torch.where(n.view(-1, 1, 1) > 0, o, 0.0)
    return out


def _noalloc(q, kv, tables, lens):
    out = torch.empty_like(q)
    B, Hkv, _ = q.shape
    kc, vc = kv[:, 0, 0], kv[:, 0, 1]
    check(lib.aeg_paged_attn_decode_noalloc(out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), kc.data_ptr(),
                                            vc.data_ptr(), kc.stride(0), kv.size(0), tables.data_ptr(), tables.stride(0),
                                            lens.data_ptr(), B, Hkv, Hkv, 128, SCALE, AEG_DTYPE_FP16,
                                            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "noalloc")
    return out


@pytest.mark.parametrize("B,Hkv,longest", [(2100, 64, 40), (1050, 128, 3)])
def test_more_pairs_than_the_scans_have_room_for(cuda_device, B, Hkv, longest):
    lens, kv, tables, q = _case(cuda_device, B, Hkv, longest, 3)
    nbytes = lib.aeg_decode_workspace_size(B, Hkv, Hkv, 128)
    area = 2 * 4096 * (8 + 4 * 128)  # partial results of two pieces a worker warp, group of one
    assert 32 * (B * Hkv + 1) > area and nbytes > area
    out = torch.empty_like(q)
    ops.read_device_errors(cuda_device)
    plan = ops.DecodePlan(B, Hkv, Hkv, 128, cuda_device).plan(lens, tables)
    ops.paged_attention_decode(out, q, kv, 0, tables, lens, SCALE, plan=plan)
    assert ops.read_device_errors(cuda_device) == 0
    want = _reference(lens, kv, tables, q)
    # fp16 outputs of weighted means: half a step of the output, 2^-11 of |v| <= 6 for P in 11 bits
    assert ((out.float() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -11 * 6).all()
    assert plan.stats()["units"] >= int((lens > 0).sum()) * Hkv
    # the same sequences in two halves, whose plans are written over the GPU: bits differ only where a sequence
    # is cut elsewhere
    half = B // 2
    for rows in (slice(0, half), slice(half, B)):
        part = torch.empty_like(q[rows])
        ops.paged_attention_decode(part, q[rows], kv, 0, tables[rows], lens[rows], SCALE)
        assert (part == out[rows]).all(-1).float().mean() > 0.9
        assert ((part.float() - want[rows]).abs() <= 2.0 ** -11 * want[rows].abs() + 2.0 ** -11 * 6).all()


@pytest.mark.parametrize("B,Hkv,longest", [(640, 62, 100), (5000, 9, 17)])
def test_both_writers_make_the_same_plan(cuda_device, B, Hkv, longest):
    """Pairs that fit a workspace's area but not the scratch's: one CTA writes the allocation-free call's lists, the
    GPU the planned call's. Same workers, same cuts: the same bits."""
    lens, kv, tables, q = _case(cuda_device, B, Hkv, longest, 4)
    assert 32 * (B * Hkv + 1) > 2 * 148 * 8 * (8 + 4 * 128) and 32 * (B * Hkv + 1) < 2 * 4096 * (8 + 4 * 128)
    ops.read_device_errors(cuda_device)
    out = torch.empty_like(q)
    ops.paged_attention_decode(out, q, kv, 0, tables, lens, SCALE)
    got = _noalloc(q, kv, tables, lens)
    assert ops.read_device_errors(cuda_device) == 0
    assert torch.equal(out, got)
    want = _reference(lens, kv, tables, q)
    assert ((out.float() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -11 * 6).all()
