"""Attention in 64 bits with a mask of any shape, and how far a kernel's results may be from it: what the tests of packed batches and of drafted trees share."""
import math

import torch

D = 128
SCALE = D ** -0.5
EPS32 = 2.0 ** -24          # half a step of a value in 32 bits
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attention64(q, k, v, seen):
    """q [Hq, S, 128], k, v [Hkv, n, 128], seen [S, n]: o, lse in 64 bits and the bounds of their errors. A row does not see what is masked, whatever it holds; one
    that sees nothing gives zeros and -inf."""
    group = q.shape[0] // k.shape[0]
    k, v = (x.double().repeat_interleave(group, 0) for x in (k, v))
    h, q64 = HALF_STEP[q.dtype], q.double()
    s = (torch.matmul(q64, k.transpose(1, 2).contiguous()) * SCALE).masked_fill_(~seen, -math.inf)
    size = torch.where(seen, torch.matmul(q64.abs(), k.abs().transpose(1, 2).contiguous()) * SCALE, 0.0)
    lse = s.logsumexp(-1)
    p = torch.where(seen, (s - lse[..., None]).exp(), 0.0)
    if v.isfinite().all():
        o, spread = p @ v, p @ v.abs()
    else:
        rows = [(i, seen[i]) for i in range(q.shape[1])]
        o = torch.stack([torch.stack([p[a, i, m] @ v[a, m] for i, m in rows]) for a in range(q.shape[0])])
        spread = torch.stack([torch.stack([p[a, i, m] @ v[a, m].abs() for i, m in rows]) for a in range(q.shape[0])])
    n = k.shape[1]
    biggest = torch.where(v.isfinite(), v, 0.0).abs().amax((1, 2))[:, None, None] if n else torch.zeros(q.shape[0], 1, 1, dtype=torch.double, device=q.device)
    # a score is a sum of 128 exact products in 32 bits: each of the 128 additions is off by half a step of at most the sum of magnitudes; the scaling adds two
    off = (size * 130 * EPS32).amax(-1) if n else torch.zeros_like(lse)
    # the exponent's argument is rounded (those that count are within 40 of the maximum), the exponential and the logarithm are off by a step
    off = off + 2.0 ** -18
    # the sum: a lane adds up its terms of every 64 keys, the lanes' sums meet
    lse_bound = 2 * off + (64 + n / 32) * EPS32 + 4 * EPS32 * lse.abs()
    # probabilities: half a step of 16 bits each, in fp16 half of 2^-24 where they are subnormal against a row sum of at least one; products of 32 keys are added up in 32
    # bits; the output: half a step, in fp16 half of 2^-24 below 2^-14
    sums = 2.0 ** -16 + n / 32 * EPS32
    o_bound = h * o.abs() + (1 + h) * ((h + 4 * off[..., None] + sums) * spread + (2.0 ** -25 * n * biggest if q.dtype == torch.float16 else 0))
    return {"o": o, "lse": lse, "o_bound": o_bound + (2.0 ** -24 if q.dtype == torch.float16 else 0.0), "lse_bound": lse_bound, "empty": ~seen.any(-1)}


def check(got_o, got_lse, want):
    """Outputs [Hq, S, 128] and [Hq, S] against what attention64 gives: infinities and NaN where it has them, zeros in rows that see nothing."""
    empty, o, lse = want["empty"], want["o"], want["lse"]
    assert (got_o[:, empty] == 0).all() and (got_lse[:, empty] == -math.inf).all()
    a, b = got_o.double()[:, ~empty], o[:, ~empty]
    fine = b.isfinite()
    assert torch.equal(a.isnan(), b.isnan()) and (a[b.isinf()] == b[b.isinf()]).all()
    far = ((a - b).abs() > want["o_bound"][:, ~empty]) & fine
    assert not far.any(), ((a - b).abs()[fine].max(), want["o_bound"][:, ~empty][fine].max())
    a, b = got_lse.double()[:, ~empty], lse[:, ~empty]
    fine = b.isfinite()
    assert torch.equal(a.isnan(), b.isnan())
    far = ((a - b).abs() > want["lse_bound"][:, ~empty]) & fine
    assert not far.any(), ((a - b).abs()[fine].max(), want["lse_bound"][:, ~empty][fine].max())
