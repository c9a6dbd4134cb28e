"""Attention of many rows (chunks of prompts) over the paged key-value cache against plain products in 64 bits: the sizes at which the work is cut in
different ways, padded batches, masked infinities and NaN, pages outside the pool, captured calls."""
import math

import pytest
import torch

import fmha_unified
from test_paged_gpu import D, EPS32, HALF_STEP, SCALE, Cache, queries

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu


def check(cache, q, o, lse, new=None, there=None):
    """`there`: per sequence, which keys are there (all). Values of keys that are there are finite."""
    B, Hq, S, _ = q.shape
    h = HALF_STEP[q.dtype]
    for b in range(B):
        n, nb = cache.seq_lens[b], S if new is None else new[b]
        if n == 0 or nb == 0:
            assert (o[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        k, v = (x.repeat_interleave(Hq // cache.Hkv, 1).transpose(0, 1).contiguous() for x in cache.keys(b))   # [Hq, n, D]
        row, key = torch.arange(S, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (key <= row + n - nb) & (row < nb)
        if there is not None:
            seen = seen & there[b].cuda()
            k, v = (torch.where(there[b].cuda()[None, :, None], x, 0.0) for x in (k, v))
        qb = q[b].double()
        s = torch.matmul(qb, k.transpose(1, 2).contiguous()) * SCALE
        # a score is a sum of 128 exact products in 32 bits: each of the 128 additions is off by half a step of at most the sum of magnitudes; the
        # scaling adds two
        size = torch.matmul(qb.abs(), k.abs().transpose(1, 2).contiguous()) * SCALE
        off = torch.where(seen, size * 130 * EPS32, 0.0).amax(-1)
        s = s.masked_fill(~seen, -math.inf)
        rl = s.logsumexp(-1)
        p = torch.where(seen, (s - rl[..., None]).exp(), 0.0)
        ro, spread = torch.matmul(p, v), torch.matmul(p, v.abs())
        biggest = torch.where(seen[None], v.abs().amax(-1)[:, None], 0.0).amax(-1)
        empty = ~seen.any(-1)
        assert (o[b][:, empty] == 0).all() and (lse[b][:, empty] == -math.inf).all()
        # the exponent's argument is rounded where it counts to 2^-18 at most; sums of n terms in blocks: 64 half steps are more than any chain's
        off = off + 2.0 ** -18
        got, want = lse[b].double()[:, ~empty], rl[:, ~empty]
        assert ((got - want).abs() <= (2 * off + 64 * EPS32)[:, ~empty] + 4 * EPS32 * want.abs()).all(), (b, (got - want).abs().max())
        # probabilities: half a step of 16 bits each, and in fp16 half of 2^-24 where they are subnormal against a row sum of at least one; the output: half
        # a step
        bound = h * ro.abs() + (1 + h) * ((h + 4 * off[..., None] + 2.0 ** -16) * spread)
        if q.dtype == torch.float16:
            bound = bound + (1 + h) * 2.0 ** -25 * n * biggest[..., None] + 2.0 ** -24
        bad = (o[b].double() - ro).abs() > bound
        assert not bad[:, ~empty].any(), (b, (o[b].double() - ro).abs().max(), bound.max())


CASES = [   # Hq, Hkv, S, page, lengths, new_lens, options
    (32, 8, 33, 32, [3000], None, {}),                                                    # a part in every workgroup
    (8, 2, 64, 16, [600, 64, 0, 1300, 40, 63], [64, 10, 64, 1, 64, 0], {}),               # a padded batch; one shorter than its rows
    (14, 2, 50, 16, [700, 1025], None, {}),                                               # 350 columns, 7 heads a row
    (3, 1, 400, 48, [4000], None, {}),
    (8, 4, 20, 16, [(97 * i) % 1100 for i in range(20)], None, {}),                       # more pairs than CUs could take in turn
    (32, 32, 130, 16, [700, 900, 130], [130, 100, 60], {}),                               # 192 triples: joined at the borders
    (32, 8, 512, 32, [1500, 513, 600, 2000], None, {}),                                   # workgroups of 256 columns
    (32, 8, 512, 32, [600] * 7 + [550], [512] * 6 + [500, 512], {}),                      # whole triples in turn, two a workgroup
    (32, 8, 128, 16, [1000, 1010, 990, 1000, 1000, 960, 1001, 999], None, {}),            # the same with two halves
    (32, 8, 1000, 32, [2000], None, {}),                                                  # one sequence, a workgroup a triple
    (64, 8, 520, 64, [700, 520, 530, 0, 1000, 600, 521, 522], None, {}),                  # more triples than are cut
    (40, 8, 65, 16, [100, 480, 65, 20], [65, 65, 3, 65], {"max_pages": 32}),              # short ones, a workgroup each
    (32, 8, 500, 32, [500], None, {}),                                                    # a prompt from its start
    (32, 8, 300, 32, [9000], None, {"token_major": True}),
    (16, 2, 8, 16, [20000, 3, 9000], None, {}),                                           # 64 columns: the other kernel's last size
    (16, 2, 9, 16, [20000, 3, 9000], None, {}),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%d-%d-S%d-p%d-B%d-%s" % (c[0], c[1], c[2], c[3], len(c[4]), max(c[4])))
def test_many_rows(gpu, case, dtype):
    Hq, Hkv, S, page, lens, new, options = case
    cache = Cache(lens, Hkv, page, dtype, **options)
    q = queries(cache, Hq, S)
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=n)
    assert o.is_contiguous() and o.shape == q.shape and o.dtype == dtype
    check(cache, q, o, lse, new)
    weights = cache.weights.clone()
    again = ops.fine_fmha_paged(q, *cache.args, new_lens=n, weights=weights)
    assert torch.equal(again, o)       # the same bits, with and without log-sum-exp and account
    other = cache.weights.clone()
    ops.fine_key_weights(q, lse, *cache.args, other, new_lens=n)
    assert torch.equal(weights.nan_to_num(7.0), other.nan_to_num(7.0))


def test_no_part_is_left_out(gpu):
    """Lengths around the edges of tiles and of the workgroups' pieces: V of ones gives ones, LSE of equal scores is s + log of their number."""
    for seed in range(14):
        gen = torch.Generator().manual_seed(seed)
        B = int(torch.randint(1, 30, (1,), generator=gen))
        Hkv, group, S = (1, 2, 8)[seed % 3], (1, 3, 4, 8)[seed % 4], (40, 70, 130, 260)[seed % 4]
        lens = (torch.rand(B, generator=gen) ** 3 * (3000 if seed % 2 else 700)).int().tolist()
        new = torch.randint(0, S + 1, (B,), generator=gen).tolist()
        cache = Cache(lens, Hkv, 16, max_pages=200 if seed % 2 else 44)
        for b, n in enumerate(lens):
            pg, sl = cache.at(b)
            cache.kv[pg, :Hkv, sl] = 0.25
            cache.kv[pg, Hkv:, sl] = 1.0
        q = torch.full((B, group * Hkv, S, D), 0.5, dtype=torch.float16, device="cuda")
        n = torch.tensor(new, dtype=torch.int32, device="cuda")
        o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=n)
        row = torch.arange(S, device="cuda")[None]
        count = torch.where(row < n[:, None], cache.lens[:, None] - n[:, None] + row + 1, 0).clamp_min(0)[:, None]   # [B, 1, S]
        assert (o == (count > 0)[..., None]).all()
        want = 0.125 * D * SCALE + count.double().log()
        assert torch.where(count > 0, (lse - want).abs() <= 4e-6, lse == -math.inf).all()


@pytest.mark.parametrize("Hq,Hkv,S,lens", [(8, 2, 64, [600, 70, 64]), (8, 8, 90, [1000, 95]), (32, 8, 80, [90, 500, 80, 100, 200])])
def test_what_a_row_does_not_see_has_no_influence_on_many(gpu, Hq, Hkv, S, lens):
    cache, clean = Cache(lens, Hkv, 16), Cache(lens, Hkv, 16)
    q = queries(cache, Hq, S)
    back = 20   # the key of the token `back` in front of the last: the rows in front of it do not see it
    for b, n in enumerate(lens):
        pg, sl = cache.at(b)
        cache.kv[pg[-1], :Hkv, sl[-1]] = float("nan")          # the last token
        cache.kv[pg[-1], Hkv:, sl[-1]] = float("inf")
        cache.kv[pg[-1 - back], Hkv:, sl[-1 - back], 5] = float("-inf")
        cache.kv[pg[-1 - back], Hkv:, sl[-1 - back], 77] = float("nan")
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
    ro, rl = ops.fine_fmha_paged_with_lse(q, *clean.args)
    for b, n in enumerate(lens):
        first = S - 1 - back   # the first row that sees that key
        front, rest = slice(0, first), slice(first, S - 1)
        # the bits can differ by the reference of the exponent, which moves with the tile's maximum: twice a row's error, |v| <= 5.5
        assert (o[b, :, front].double() - ro[b, :, front].double()).abs().max() <= 4 * 2.0 ** -11 * 5.5
        assert (lse[b, :, :S - 1] - rl[b, :, :S - 1]).abs().max() <= 1e-5
        others = [d for d in range(D) if d not in (5, 77)]
        assert (o[b][:, rest][..., others].double() - ro[b][:, rest][..., others].double()).abs().max() <= 4 * 2.0 ** -11 * 5.5
        # (a probability that is rounded to nothing makes NaN of an infinity)
        assert ((o[b, :, rest, 5] == -math.inf) | o[b, :, rest, 5].isnan()).all() and (o[b, :, first, 5] == -math.inf).any()
        assert o[b, :, rest, 77].isnan().all()
        assert o[b, :, -1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("S", [40, 200])
def test_pages_outside_the_pool_hold_no_keys_for_many_rows(gpu, S, dtype):
    lens = [1300, 700, 208]
    cache = Cache(lens, 2, 32, dtype)
    q = queries(cache, 8, S)
    outside = {0: [2, 30, 31], 1: [0, 21], 2: list(range(7))}
    there = []
    for b, n in enumerate(lens):
        for i in outside[b]:
            cache.table[b, i] = (-1, cache.kv.shape[0], 2 ** 31 - 1, -2 ** 31)[i % 4]
        there.append(~torch.isin(torch.arange(n) // 32, torch.tensor(outside[b])))
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
    table = cache.table.clone()
    cache.table.clamp_(0, cache.kv.shape[0] - 1)    # (for the oracle, which leaves those keys out)
    for b, n in enumerate(lens):
        assert int(there[b].sum()) == n - sum(min(32, n - 32 * i) for i in outside[b])
    check(cache, q, o, lse, None, there)
    cache.table.copy_(table)


def test_a_captured_chunk_serves_the_lengths_it_finds(gpu):
    cache = Cache([3000, 1200, 900, 64], 8, 32)
    S = 96
    q = queries(cache, 32, S)
    new = torch.full((4,), S, dtype=torch.int32, device="cuda")
    eager = ops.fine_fmha_paged(q, *cache.args, new_lens=new)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=new)
    for lens, rows in (([3000, 1200, 900, 64], [S] * 4), ([0, 1, 97, 3000 % 64], [S, 1, S, 7]), ([2999, 0, 96, 33], [S, 0, 50, S]), ([3000, 1200, 900, 64], [S] * 4)):
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        new.copy_(torch.tensor(rows, dtype=torch.int32))
        g.replay()
        o, l = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=new)
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(lse, l)
    assert torch.equal(out, eager)


def test_chunks_on_two_streams_at_once(gpu):
    caches = [Cache([2000, 300], 8, 32, seed=s) for s in (1, 2)]
    qs = [queries(c, 32, 150, seed=s) for s, c in enumerate(caches)]
    alone = [ops.fine_fmha_paged(q, *c.args) for q, c in zip(qs, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(ops.fine_fmha_paged(qs[k], *caches[k].args))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, alone[k]) for o in got[k])


@pytest.mark.parametrize("Hq,Hkv,S,lens,new", [(32, 1, 2049, [2100], None), (64, 2, 2100, [2100, 2300], [2001, 2100])])
def test_more_than_65535_columns(gpu, Hq, Hkv, S, lens, new):
    """2049 rows of 32 query heads on a kv head: what the rows see, and the account from the scores worked out again."""
    cache = Cache(lens, Hkv, 32)
    q = queries(cache, Hq, S)
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    before = cache.weights.clone()
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=n, weights=cache.weights)
    check(cache, q, o, lse, new)
    again = before.clone()
    ops.fine_key_weights(q, lse, *cache.args, again, new_lens=n)
    assert torch.equal(again.nan_to_num(7.0), cache.weights.nan_to_num(7.0))
    for b, length in enumerate(lens):
        pg, sl = cache.at(b)
        rows = S if new is None else new[b]
        total = (cache.weights[pg, :, sl].double() - before[pg, :, sl].double()).sum(0)
        # each row's probabilities sum to one: a score is off by 130 half steps of sums of magnitudes of 128 |q| |k| / 11.3 <= 60, the LSE as much, the account's
        # additions by 2^-24 of values up to Hq / Hkv * rows a step
        count = Hq // Hkv * rows
        assert ((total - count).abs() <= count * (2 * 130 * 60 * EPS32 + 2.0 ** -16)).all()


def test_the_last_rows_of_a_prompt_of_any_length_count(gpu):
    Hq, Hkv, S, last = 32, 8, 16500, 64
    cache = Cache([S], Hkv, 64)
    q = queries(cache, Hq, last)
    whole = torch.full((1, Hq, S, D), math.nan, dtype=torch.float16, device="cuda")
    whole[:, :, -last:] = q
    _, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
    wide = torch.full((1, Hq, S), math.nan, device="cuda")
    wide[:, :, -last:] = lse
    a, b = cache.weights.clone(), cache.weights.clone()
    ops.fine_key_weights(whole, wide, *cache.args, a, last_rows=last)
    ops.fine_key_weights(q, lse, *cache.args, b)
    assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
