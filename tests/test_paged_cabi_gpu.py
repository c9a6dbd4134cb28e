"""The C entry points of the paged key-value cache, called as a C program calls them: the structure filled from addresses and strides, the caller's
workspace, strides left out. They give the bits of the operators in `fmha_unified.ops`, whose results other tests hold against plain loops."""
import ctypes

import pytest
import torch

import fmha_unified
import mi355_serving as lib

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu
D = 128
SCALE = D ** -0.5


def pool(dtype, lens, Hkv=2, page=16):
    """A pool with two heads that no kv head has between the pages, so that no stride is the dense one."""
    gen = torch.Generator().manual_seed(11)
    pages = [-(-n // page) for n in lens]
    wide = torch.randn(sum(pages) + 3, 2 * Hkv + 2, page, D, generator=gen).to(dtype).cuda()
    order = torch.randperm(sum(pages) + 3, generator=gen).int()
    table = torch.full((len(lens), max(pages) + 2), -1, dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = order[sum(pages[:b]):sum(pages[:b]) + n]
    weights = torch.rand(len(wide), Hkv, page, generator=gen).cuda()
    positions = torch.randint(0, 5000, (len(wide), Hkv, page), generator=gen, dtype=torch.int32).cuda()
    return wide[:, :2 * Hkv], table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), weights, positions


def ptr(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def workspace(size):
    """What the library asked for, full of NaN: its contents are irrelevant."""
    return torch.full((size,), 255, dtype=torch.uint8, device="cuda") if size else None


def run(entry, *args):
    code = entry(*args)
    assert code == 0, (code, lib.load().mi355_last_error())


@pytest.mark.parametrize("S", [1, 3, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attention_and_what_prompts_attended_to(gpu, dtype, S):
    c = lib.load()
    kv, table, lens, weights, _ = pool(dtype, [300, 40, 1900])
    B, Hq = 3, 8
    q = torch.randn(B, Hq, S, D, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    new = torch.tensor([S, max(S - 1, 1), S], dtype=torch.int32, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    theirs = weights.clone()
    cache = lib.paged_kv(kv, table, lens, new, weights)
    o, lse = torch.empty_like(q), torch.empty(B, Hq, S, device="cuda")
    size = c.mi355_fmha_paged_workspace_bytes(ctypes.byref(cache), Hq, S, 1)
    ws = workspace(size)
    run(c.mi355_fmha_paged, ctypes.byref(cache), ptr(q), ptr(o), ptr(lse), Hq, S, None, SCALE, ptr(ws), size, stream)
    want_o, want_lse = ops.fine_fmha_paged_with_lse(q, kv, table, lens, new, theirs)
    assert torch.equal(o, want_o) and torch.equal(lse, want_lse) and torch.equal(weights, theirs)
    size = c.mi355_fmha_key_weights_workspace_bytes(ctypes.byref(cache), Hq, S, 0)
    ws = workspace(size)
    run(c.mi355_fmha_key_weights, ctypes.byref(cache), ptr(q), ptr(lse), Hq, S, None, 0, SCALE, ptr(ws), size, stream)
    ops.fine_key_weights(q, lse, kv, table, lens, theirs, new)
    assert torch.equal(weights, theirs)
    # one byte less than was asked for is refused, and nothing runs
    if size:
        assert c.mi355_fmha_key_weights(ctypes.byref(cache), ptr(q), ptr(lse), Hq, S, None, 0, SCALE, ptr(ws), size - 1, stream) == lib.ERR_BAD_ARGUMENT
        assert torch.equal(weights, theirs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_filing_and_eviction(gpu, dtype):
    c = lib.load()
    kv, table, lens, weights, positions = pool(dtype, [300, 40, 1900])
    B, Hq, Hkv, S = 3, 4, 2, 5
    mine = (kv.clone(), weights.clone(), positions.clone())
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=gen).to(dtype).cuda()
    x = qkv.clone()
    cos, sin = torch.randn(50, 64, generator=gen).cuda(), torch.randn(50, 64, generator=gen).cuda()
    at = torch.randint(0, 50, (B, S), generator=gen, dtype=torch.int32).cuda()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    cache = lib.paged_kv(mine[0], table, lens, None, mine[1], mine[2])
    run(c.mi355_rope_paged, ctypes.byref(cache), ptr(x), S, Hq, 1, x.stride(0), x.stride(1), ptr(cos), ptr(sin), ptr(at), S, 50, stream)
    ops.fine_rope_paged(qkv, kv, table, lens, cos, sin, at, Hq, weights=weights, key_positions=positions, keep_keys=True)
    assert torch.equal(x, qkv) and torch.equal(mine[0], kv) and torch.equal(mine[1], weights) and torch.equal(mine[2], positions)
    out = torch.empty_like(lens)
    size = c.mi355_cache_evict_workspace_bytes(ctypes.byref(cache), 128)
    ws = workspace(size)
    run(c.mi355_cache_evict, ctypes.byref(cache), 128, 32, ptr(out), ptr(ws), size, stream)
    left = ops.fine_evict_paged(kv, table, lens, weights, positions, 128, 32)
    assert torch.equal(out, left) and out.tolist() == [128, 40, 128]
    assert torch.equal(mine[0], kv) and torch.equal(mine[1], weights) and torch.equal(mine[2], positions)


@pytest.mark.parametrize("S", [2, 40])
def test_scales_of_every_size(gpu, S):
    """From one that makes all scores alike (the mean of the values that a row sees) to one that leaves the largest score alone."""
    c = lib.load()
    kv, table, lens, _, _ = pool(torch.float16, [700, 60])
    B, Hq, Hkv, page = 2, 8, 2, 16
    q = torch.randn(B, Hq, S, D, generator=torch.Generator().manual_seed(4)).half().cuda()
    cache = lib.paged_kv(kv, table, lens)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    size = c.mi355_fmha_paged_workspace_bytes(ctypes.byref(cache), Hq, S, 1)
    for scale in (1e-38, 1e-30, 1e-6, 50.0, 1e6):
        o, lse, ws = torch.empty_like(q), torch.empty(B, Hq, S, device="cuda"), workspace(size)
        run(c.mi355_fmha_paged, ctypes.byref(cache), ptr(q), ptr(o), ptr(lse), Hq, S, None, scale, ptr(ws), size, stream)
        for b, n in enumerate([700, 60]):
            j = torch.arange(n, device="cuda")
            x = kv[table[b].long()[j // page], :, j % page].double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)   # [2 Hq, n, D]
            s = torch.matmul(q[b].double(), x[:Hq].transpose(1, 2).contiguous())
            seen = j[None] <= torch.arange(S, device="cuda")[:, None] + n - S
            if scale < 1e-5:   # the largest |score| is below 80: probabilities are alike but for 1.6e-4 of themselves, rounded to 16 bits (2^-11), and so is their mean
                mean = torch.matmul(seen.double(), x[Hq:]) / seen.sum(1)[:, None]
                spread = torch.matmul(seen.double(), x[Hq:].abs()) / seen.sum(1)[:, None]
                assert ((o[b].double() - mean).abs() <= (2 * 2.0 ** -11 + 2e-4) * spread + 2.0 ** -11 * mean.abs() + 2.0 ** -24).all()
                assert ((lse[b].double() - seen.sum(1).double().log()).abs() <= 2e-4).all()
            else:              # rows whose two largest scores are more than 25 apart, after scaling, have the value of the first: the others have e^-25 n of the sum
                top = torch.where(seen, s, -1e30).topk(2, -1)
                alone = (top.values[..., 0] - top.values[..., 1]) * scale > 25
                first = torch.gather(x[Hq:], 1, top.indices[..., :1].expand(-1, -1, D))
                assert alone.float().mean() > 0.5
                # its probability is 2^x against the exponent's reference, which may be any of the row's maxima so far (x up to 8): rounded to 16 bits in the
                # product (2^-11), not in the sum; the quotient is rounded once more (2^-11)
                assert ((o[b].double() - first).abs() <= 2.001 * 2.0 ** -11 * first.abs() + 1e-6)[alone].all()
                assert torch.isfinite(o[b]).all()
