"""The paged key-value cache against plain loops in 64 bits: attention over pages, filing, what prompts attended to, eviction, and a run of
them as a generation loop makes it."""
import math

import pytest
import torch

import fmha_unified

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu
D = 128
SCALE = D ** -0.5
EPS32 = 2.0 ** -24          # half a step of a value in 32 bits
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Cache:
    """A pool whose pages are handed out at random. Everything that holds no key is NaN (or a position that nothing has)."""

    def __init__(self, seq_lens, Hkv, page, dtype=torch.float16, spare=2, seed=0, max_pages=None, token_major=False, scale=1.0):
        self.gen = torch.Generator().manual_seed(seed)
        B = len(seq_lens)
        P = max_pages or max(1, max(-(-n // page) for n in seq_lens))
        n_pages = sum(-(-n // page) for n in seq_lens) + spare
        shape = (n_pages, 2 * Hkv, page, D)
        if token_major:
            self.kv = torch.full((n_pages, page, 2 * Hkv + 1, D), float("nan"), dtype=dtype, device="cuda")[:, :, :2 * Hkv].transpose(1, 2)
        else:
            self.kv = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        order = torch.randperm(n_pages, generator=self.gen).tolist()
        table = torch.full((B, P), -7, dtype=torch.int32)
        for b, n in enumerate(seq_lens):
            for i in range(-(-n // page)):
                table[b, i] = order.pop()
        self.table = table.cuda()
        self.lens = torch.tensor(seq_lens, dtype=torch.int32, device="cuda")
        self.seq_lens, self.page, self.Hkv, self.dtype = list(seq_lens), page, Hkv, dtype
        self.weights = torch.full((n_pages, Hkv, page), float("nan"), device="cuda")
        self.positions = torch.full((n_pages, Hkv, page), -12345, dtype=torch.int32, device="cuda")
        for b, n in enumerate(seq_lens):
            pg, sl = self.at(b, n)
            self.kv[pg, :, sl] = (torch.randn(n, 2 * Hkv, D, generator=self.gen) * scale).to(dtype).cuda()
            self.weights[pg, :, sl] = torch.rand(n, Hkv, generator=self.gen).cuda()

    def at(self, b, n=None, table=None):
        j = torch.arange(self.seq_lens[b] if n is None else n)
        return (self.table if table is None else table)[b].cpu().long()[j // self.page].cuda(), (j % self.page).cuda()

    def keys(self, b):
        """K, V [n, Hkv, 128] in 64 bits."""
        pg, sl = self.at(b)
        x = self.kv[pg, :, sl].double()
        return x[:, :self.Hkv], x[:, self.Hkv:]

    args = property(lambda self: (self.kv, self.table, self.lens))


def reference(cache, q, new, b):
    """O, LSE, p [Hq, S, n] and what bounds their errors, of sequence b, in 64 bits."""
    Hq, S = q.shape[1:3]
    n = cache.seq_lens[b]
    k, v = cache.keys(b)
    group = Hq // cache.Hkv
    k, v = k.repeat_interleave(group, 1).transpose(0, 1), v.repeat_interleave(group, 1).transpose(0, 1)   # [Hq, n, D]
    s = torch.matmul(q[b].double(), k.transpose(1, 2).contiguous()) * SCALE
    size = torch.matmul(q[b].double().abs(), k.abs().transpose(1, 2).contiguous()) * SCALE
    row, key = torch.arange(S, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (key <= row + n - new) & (row < new)
    s = s.masked_fill(~seen, -math.inf)
    lse = s.logsumexp(-1)
    p = torch.where(seen, (s - lse[..., None]).exp(), 0.0)
    # a row does not see what is masked, whatever it holds
    o = torch.stack([torch.stack([p[h, i, seen[i]] @ v[h, seen[i]] for i in range(S)]) for h in range(Hq)])
    spread = torch.stack([torch.stack([p[h, i, seen[i]] @ v[h, seen[i]].abs() for i in range(S)]) for h in range(Hq)])
    biggest = torch.where(seen[None, :, :, None], v.abs()[:, None], 0.0).amax((2, 3)) if n else torch.zeros(Hq, S, dtype=torch.double, device="cuda")
    # a score is a sum of 128 exact products in 32 bits: each of the 128 additions is off by half a step of at most the sum of magnitudes; the scaling adds two
    off_s = torch.where(seen, size * 130 * EPS32, 0.0).amax(-1) if n else torch.zeros(Hq, S, dtype=torch.double, device="cuda")
    return o, lse, p, seen, spread, biggest, off_s


def check_attention(cache, q, o, lse, new=None, weights_before=None):
    B, Hq, S, _ = q.shape
    for b in range(B):
        nb = S if new is None else new[b]
        n = cache.seq_lens[b]
        ro, rl, p, seen, spread, biggest, off_s = reference(cache, q, nb, b)
        empty = ~seen.any(-1)
        assert (o[b][:, empty] == 0).all() and (lse[b][:, empty] == -math.inf).all()
        # the exponent's argument is rounded (values up to |s| + |reference| <= 2 * 150 / ln 2 would be off by 2^-16; those that count are within
        # 40 of the maximum), the exponential and the logarithm are off by a step, the sum of n terms by n half steps at most in any order,
        # in blocks: 64 is more than the length of any chain here times two
        off = off_s + 2.0 ** -18
        got, want = lse[b].double()[:, ~empty], rl[:, ~empty]
        assert ((got - want).abs() <= (2 * off + 64 * EPS32)[:, ~empty] + 4 * EPS32 * want.abs()).all()
        # probabilities: half a step of 16 bits each, and in fp16 half of 2^-24 where they are subnormal against a row sum of at least one; the output: half
        # a step
        h = HALF_STEP[q.dtype]
        bound = h * ro.abs() + (1 + h) * ((h + 4 * off[..., None] + 2.0 ** -16) * spread + (2.0 ** -25 * n * biggest[..., None] if q.dtype == torch.float16 else 0))
        tiny = 2.0 ** -24 if q.dtype == torch.float16 else 0.0   # an fp16 result below 2^-14
        bad = (o[b].double() - ro).abs() > bound + tiny
        assert not bad[:, ~empty].any(), (b, (o[b].double() - ro).abs().max(), bound.max())
        if weights_before is not None:
            pg, sl = cache.at(b)
            before, after = weights_before[pg, :, sl].double(), cache.weights[pg, :, sl].double()       # [n, Hkv]
            add = p.unflatten(0, (cache.Hkv, -1)).sum((1, 2)).T
            slack = (p * (4 * off + 2.0 ** -18)[..., None]).unflatten(0, (cache.Hkv, -1)).sum((1, 2)).T
            terms = Hq // cache.Hkv * S
            assert ((after - before - add).abs() <= slack + EPS32 * after.abs() * 2 + terms * EPS32 * add + 1e-30).all()
    if weights_before is not None:   # nothing else has changed
        there = torch.zeros(cache.weights.shape, dtype=torch.bool, device="cuda")
        for b in range(B):
            pg, sl = cache.at(b)
            there[pg, :, sl] = True
        same = cache.weights == weights_before
        assert (same | there | (cache.weights.isnan() & weights_before.isnan())).all()


def queries(cache, Hq, S, seed=1, scale=1.5):
    gen = torch.Generator().manual_seed(seed)
    B = len(cache.seq_lens)
    return (torch.randn(B, S, Hq, D, generator=gen) * scale).to(cache.dtype).cuda().transpose(1, 2)


ATTENTION = [   # Hq, Hkv, S, page, lengths, new_lens, options
    (8, 2, 1, 16, [300], None, {}),
    (8, 2, 1, 16, [1, 15, 16, 17, 0, 31, 32, 33], None, {}),
    (32, 8, 1, 64, [8191], None, {}),
    (32, 8, 1, 16, [8192, 1, 0, 513, 4097, 31], None, {}),
    (64, 8, 1, 48, [1000, 1023, 0, 2049], None, {}),
    (32, 32, 1, 128, [700, 512], None, {}),
    (40, 8, 2, 32, [600, 1500, 2], None, {}),
    (1, 1, 1, 16, [5000], None, {}),
    (6, 2, 3, 16, [2, 40, 700, 0, 3], None, {}),                        # shorter than their rows
    (32, 8, 4, 32, [900, 33, 700, 64], [4, 1, 0, 3], {}),               # a padded batch
    (64, 8, 4, 16, [513, 1025], None, {}),                              # 32 columns
    (16, 2, 7, 32, [800, 77], [7, 5], {}),                              # 56 columns: two blocks
    (8, 2, 100, 16, [100, 731], [100, 66], {}),                         # a chunk of a prompt
    (32, 8, 1, 16, [512] * 2, None, {"max_pages": 32}),                 # the longest that one workgroup walks
    (32, 8, 1, 16, [300, 20], None, {"max_pages": 900}),                # a table much longer than its sequences
    (8, 4, 1, 16, [(37 * i) % 97 for i in range(70)], None, {}),        # more than 64 sequences
    (8, 1, 1, 32, [(537 * i) % 1997 for i in range(130)], None, {}),
    (32, 8, 1, 32, [1025, 7], None, {"token_major": True}),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("account", [False, True], ids=["plain", "account"])
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "%d-%d-S%d-p%d-B%d-%s" % (c[0], c[1], c[2], c[3], len(c[4]), max(c[4])))
def test_attention_over_pages(gpu, case, account, dtype):
    Hq, Hkv, S, page, lens, new, options = case
    cache = Cache(lens, Hkv, page, dtype, **options)
    q = queries(cache, Hq, S)
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    before = cache.weights.clone()
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=n, weights=cache.weights if account else None)
    assert o.is_contiguous() and o.shape == q.shape and o.dtype == dtype
    check_attention(cache, q, o, lse, new, before if account else None)
    again = ops.fine_fmha_paged(q, *cache.args, new_lens=n, weights=before if account else None)
    assert torch.equal(again, o)       # the same bits, with and without the log-sum-exp
    if account:
        assert torch.equal(before.nan_to_num(7.0), cache.weights.nan_to_num(7.0))


def test_the_cut_of_the_work_leaves_nothing_out(gpu):
    """Lengths around every edge of the tiles and of the workgroups' shares: V of ones gives ones, LSE of equal scores is s + log n."""
    for seed in range(12):
        gen = torch.Generator().manual_seed(seed)
        B = int(torch.randint(1, 90, (1,), generator=gen))
        lens = (torch.rand(B, generator=gen) ** 3 * 3000).int().tolist()
        Hkv = (1, 2, 8)[seed % 3]
        cache = Cache(lens, Hkv, 16, max_pages=200)
        for b, n in enumerate(lens):
            pg, sl = cache.at(b)
            cache.kv[pg, :Hkv, sl] = 0.25
            cache.kv[pg, Hkv:, sl] = 1.0
        q = torch.full((B, 2 * Hkv, 1, D), 0.5, dtype=torch.float16, device="cuda")
        o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
        n = cache.lens.double()[:, None, None]
        assert (o == (n > 0)[..., None]).all()
        want = 0.125 * D * SCALE + n.log()
        assert torch.where(n > 0, (lse - want).abs() <= 4e-6, lse == -math.inf).all()


def test_what_a_row_does_not_see_has_no_influence(gpu):
    """Infinities and NaN in keys and values that are masked for some rows, and in pages outside the pool."""
    for S, lens, page in ((4, [600, 70, 5], 16), (3, [1500], 32), (4, [4], 16)):
        cache = Cache(lens, 2, page)
        q = queries(cache, 8, S)
        for b, n in enumerate(lens):   # the last token's key and value: the rows in front of it do not see them
            pg, sl = cache.at(b)
            cache.kv[pg[-1], :2, sl[-1]] = float("nan")
            cache.kv[pg[-1], 2:, sl[-1]] = float("inf")
        clean = Cache(lens, 2, page)
        o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
        ro, rl = ops.fine_fmha_paged_with_lse(q, *clean.args)
        assert torch.isfinite(o[:, :, :-1]).all()
        # the kept rows' values (the last bits: a NaN score leaves the reference of the exponent to the others)
        assert (o[:, :, :-1].double() - ro[:, :, :-1].double()).abs().max() <= 4 * 2.0 ** -11 * 5
        assert (lse[:, :, :-1] - rl[:, :, :-1]).abs().max() <= 1e-5
        assert o[:, :, -1].isnan().all()


@pytest.mark.parametrize("S,lens", [(4, [300]), (4, [5000, 70]), (3, [40, 1]), (40, [900])])
def test_a_row_of_nan_leaves_the_account_of_keys_that_it_does_not_see(gpu, S, lens):
    cache = Cache(lens, 2, 16)
    q = queries(cache, 8, S)
    w, want = cache.weights.clone(), cache.weights.clone()
    ops.fine_fmha_paged_with_lse(q, *cache.args, weights=want)
    q[:, :, 0] = math.nan
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, weights=w)
    for b, n in enumerate(lens):
        pg, sl = cache.at(b)
        seen = max(n - S + 1, 0)                                   # keys of the first row
        assert o[b, :, 0].isnan().all() if seen else (o[b, :, 0] == 0).all()
        assert torch.isfinite(o[b, :, max(S - n, 0) + (seen > 0):]).all()
        assert w[pg[:seen], :, sl[:seen]].isnan().all()
        # of the others' sums, up to 160 probabilities of at most one: the exponent's reference may be another one, which moves each by 2^-16 of itself
        got, ref = w[pg[seen:], :, sl[seen:]], want[pg[seen:], :, sl[seen:]]
        assert ((got - ref).abs() <= 160 * 2.0 ** -16).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_pages_outside_the_pool_hold_no_keys(gpu, dtype):
    lens = [300, 700, 64]
    cache = Cache(lens, 2, 32, dtype)
    q = queries(cache, 8, 1)
    full = cache.table.clone()
    cache.table[0, 2] = -1
    cache.table[1, 0] = cache.kv.shape[0]
    cache.table[1, 21] = 2 ** 31 - 1
    cache.table[2] = -2 ** 31
    before = cache.weights.clone()
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args, weights=cache.weights)
    # the same keys without those pages
    left = [[i for i in range(-(-n // 32)) if 0 <= int(cache.table[b, i]) < cache.kv.shape[0]] for b, n in enumerate(lens)]
    short = [sum(min(32, n - 32 * i) for i in left[b]) for b, n in enumerate(lens)]
    other = Cache(lens, 2, 32, dtype)
    other.kv, other.weights, other.seq_lens = cache.kv, cache.weights, short
    other.lens = torch.tensor(short, dtype=torch.int32, device="cuda")
    other.table = torch.full_like(full, -1)
    for b in range(3):
        for j, i in enumerate(left[b]):
            other.table[b, j] = full[b, i]
    check_attention(other, q, o, lse, None, before)
    # filing and the prompt's account leave them alone too
    kv, w = cache.kv.clone(), cache.weights.clone()
    qkv = torch.randn(3, 40, 12, D, device="cuda").to(dtype)
    ones = torch.ones(50, 64, device="cuda")
    cache.table[:] = -1
    ops.fine_rope_paged(qkv, *cache.args, ones, ones, torch.arange(40, dtype=torch.int32, device="cuda"), 8, weights=cache.weights)
    ops.fine_key_weights(qkv[:, :, :8].transpose(1, 2), torch.zeros(3, 8, 40, device="cuda"), *cache.args, cache.weights)
    lens_out = ops.fine_evict_paged(*cache.args, cache.weights, cache.positions, 50, 10)
    assert torch.equal(kv.nan_to_num(7.0), cache.kv.nan_to_num(7.0)) and torch.equal(w.nan_to_num(7.0), cache.weights.nan_to_num(7.0))
    assert lens_out.tolist() == [50, 50, 50]


def test_lengths_beyond_the_table_are_cut(gpu):
    cache = Cache([640, 100], 2, 16)
    q = queries(cache, 8, 1)
    want = ops.fine_fmha_paged(q, *cache.args)
    cache.lens[0] = 2 ** 31 - 1
    cache.lens[1] = -5
    o, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
    assert torch.equal(o[0], want[0]) and (o[1] == 0).all() and (lse[1] == -math.inf).all()


def test_pages_far_into_a_large_pool(gpu):
    """Addresses beyond 2^32 bytes and element offsets beyond 2^31: a pool of pages 1.5 GiB apart."""
    stride = 3 << 28   # elements
    store = torch.empty(5 * stride, dtype=torch.float16, device="cuda")
    cache = Cache([70, 33], 2, 32, spare=0)   # five pages
    kv = store.as_strided((5, 4, 32, D), (stride, 32 * D, D, 1))
    kv.copy_(cache.kv)
    assert cache.kv.shape[0] == 5
    q = queries(cache, 8, 1)
    assert torch.equal(ops.fine_fmha_paged(q, kv, cache.table, cache.lens), ops.fine_fmha_paged(q, *cache.args))
    w = cache.weights[:5].contiguous()
    lse = torch.zeros(2, 8, 1, device="cuda")
    w1, w2 = w.clone(), cache.weights.clone()
    ops.fine_key_weights(q, lse, kv, cache.table, cache.lens, w1)
    ops.fine_key_weights(q, lse, *cache.args, w2)
    assert torch.equal(w1.nan_to_num(7.0), w2[:5].nan_to_num(7.0))
    pos = torch.arange(5 * 2 * 32, dtype=torch.int32, device="cuda").reshape(5, 2, 32)
    near = kv.clone()
    p1, p2 = pos.clone(), pos.clone()
    w2 = w1.clone()
    a = ops.fine_evict_paged(kv, cache.table, cache.lens, w1, p1, 30, 5)
    b = ops.fine_evict_paged(near, cache.table, cache.lens, w2, p2, 30, 5)
    assert torch.equal(a, b) and torch.equal(p1, p2) and torch.equal(kv.nan_to_num(7.0), near.nan_to_num(7.0))
    qkv = torch.randn(2, 3, 12, D, device="cuda", dtype=torch.float16)
    t = torch.rand(50, 64, device="cuda")
    for pool in (kv, near):
        ops.fine_rope_paged(qkv.clone(), pool, cache.table, cache.lens, t, t, torch.arange(3, dtype=torch.int32, device="cuda"), 8)
    assert torch.equal(kv.nan_to_num(7.0), near.nan_to_num(7.0))


# ---- filing ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,S,page,lens,new,keep,shared", [
    (32, 8, 1, 16, [1, 16, 17, 4096], None, False, False),
    (8, 2, 5, 16, [5, 20, 3, 0, 40], [5, 3, 4, 0, 1], False, False),      # the third brings more tokens than it is long
    (32, 8, 130, 64, [130, 200], None, True, True),
    (40, 8, 33, 48, [33, 90], [33, 20], True, False),
    (0, 1, 3, 32, [70], None, False, False),                              # nothing but a key and a value head
])
def test_filing_of_new_tokens(gpu, Hq, Hkv, S, page, lens, new, keep, shared, dtype):
    B, heads = len(lens), Hq + 2 * Hkv
    cache = Cache(lens, Hkv, page, dtype)
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(B, S, heads + 2, D, generator=gen).to(dtype).cuda()
    qkv = wide[:, :, :heads]                                              # a row longer than its heads
    angle = torch.arange(5000, dtype=torch.double)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.double) / 64)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    positions = torch.randint(0, 5000, (S,) if shared else (B, S), generator=gen, dtype=torch.int32).cuda()
    x, kv, w, pos = wide.clone(), cache.kv.clone(), cache.weights.clone(), cache.positions.clone()
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    ops.fine_rope_paged(qkv, *cache.args, cos, sin, positions, Hq, new_lens=n, weights=cache.weights, key_positions=cache.positions, keep_keys=keep)
    h = HALF_STEP[dtype]
    where = positions.expand(B, S) if shared else positions
    for b in range(B):
        nb = S if new is None else new[b]
        for t in range(S):
            if t >= nb:
                assert torch.equal(wide[b, t], x[b, t])
                continue
            p = int(where[b, t])
            c, s = cos[p].double(), sin[p].double()
            old = x[b, t, :Hq + Hkv].double()
            lo, hi = old[..., :64], old[..., 64:]
            want = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
            room = h * want.abs() + 4 * EPS32 * torch.cat((lo.abs() * c.abs() + hi.abs() * s.abs(), hi.abs() * c.abs() + lo.abs() * s.abs()), -1) + 2.0 ** -25
            assert ((wide[b, t, :Hq].double() - want[:Hq]).abs() <= room[:Hq]).all()
            if keep:
                assert ((wide[b, t, Hq:Hq + Hkv].double() - want[Hq:]).abs() <= room[Hq:]).all()
            else:
                assert torch.equal(wide[b, t, Hq:Hq + Hkv], x[b, t, Hq:Hq + Hkv])
            assert torch.equal(wide[b, t, Hq + Hkv:], x[b, t, Hq + Hkv:])
            key = lens[b] - nb + t
            if key < 0:
                continue
            pg, sl = int(cache.table[b, key // page]), key % page
            assert ((cache.kv[pg, :Hkv, sl].double() - want[Hq:]).abs() <= room[Hq:]).all()
            assert torch.equal(cache.kv[pg, Hkv:, sl], x[b, t, Hq + Hkv:heads])
            assert (cache.weights[pg, :, sl] == 0).all() and (cache.positions[pg, :, sl] == p).all()
            if keep:
                assert torch.equal(cache.kv[pg, :Hkv, sl], wide[b, t, Hq:Hq + Hkv])
            # as they were, for what follows
            cache.kv[pg, :, sl], cache.weights[pg, :, sl], cache.positions[pg, :, sl] = kv[pg, :, sl], w[pg, :, sl], pos[pg, :, sl]
    for got, was in ((cache.kv, kv), (cache.weights, w), (cache.positions, pos)):
        assert torch.equal(got.nan_to_num(7.0), was.nan_to_num(7.0))


def test_filing_is_the_contiguous_caches_arithmetic(gpu):
    """Bit for bit what mi355_rope_qkv does."""
    import mi355_serving as lib
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 20, 12, D, generator=gen).half().cuda()
    angle = torch.arange(64, dtype=torch.double)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.double) / 64)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    pos = torch.arange(20, dtype=torch.int32, device="cuda")
    dense = torch.zeros(2, 4, 20, D, dtype=torch.float16, device="cuda")
    a, b = qkv.clone(), qkv.clone()
    lib.rope_qkv(a, dense.transpose(1, 2), cos, sin, pos, 8, 2)
    cache = Cache([20, 20], 2, 16)
    ops.fine_rope_paged(b, *cache.args, cos, sin, pos, 8)
    assert torch.equal(a[:, :, :8], b[:, :, :8])
    for i in range(2):
        pg, sl = cache.at(i)
        assert torch.equal(cache.kv[pg, :, sl], dense[i].transpose(0, 1))


# ---- what prompts attended to --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,S,page,lens,new,last", [
    (8, 2, 1, 16, [1], None, 0),
    (8, 2, 17, 16, [17, 300], None, 0),
    (32, 8, 64, 48, [2050], None, 0),
    (4, 1, 700, 16, [700, 257], [700, 257], 0),
    (4, 4, 600, 32, [1111, 600, 5], [600, 64, 5], 32),
    (6, 2, 130, 128, [130, 0, 100, 40], [130, 0, 130, 20], 0),            # one shorter than its rows
    (2, 1, 1500, 16, [1500], None, 0),
    (2, 1, 300, 16, [300], None, 1),
    (2, 1, 300, 16, [300], None, 1000),
])
def test_what_a_prompt_attended_to(gpu, Hq, Hkv, S, page, lens, new, last, dtype):
    cache = Cache(lens, Hkv, page, dtype)
    q = queries(cache, Hq, S)
    B = len(lens)
    refs = [reference(cache, q, S if new is None else new[b], b) for b in range(B)]
    lse = torch.stack([r[1] for r in refs]).float()
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    before = cache.weights.clone()
    ops.fine_key_weights(q, lse, *cache.args, cache.weights, new_lens=n, last_rows=last)
    first = cache.weights.clone()
    for b in range(B):
        nb = S if new is None else new[b]
        _, rl, p, seen, _, _, off_s = refs[b]
        if last:
            p = p.clone()
            p[:, :max(0, nb - last)] = 0
        # the LSE that the kernel is given is rounded
        off = off_s + 2.0 ** -18 + EPS32 * torch.where(rl.isinf(), 0.0, rl.abs())
        pg, sl = cache.at(b)
        add = p.unflatten(0, (Hkv, -1)).sum((1, 2)).T
        slack = (p * (2 * off)[..., None]).unflatten(0, (Hkv, -1)).sum((1, 2)).T
        got = first[pg, :, sl].double() - before[pg, :, sl].double()
        # sums of up to Hq / Hkv * S terms, in chains of at most 4 a tile, 16 lanes and the ranges
        chain = 4 * (Hq // Hkv) * (S // 64 + 1) + 16
        assert ((got - add).abs() <= slack + chain * EPS32 * add + 2 * EPS32 * first[pg, :, sl].double().abs() + 1e-30).all(), b
    cache.weights.copy_(before)
    ops.fine_key_weights(q, lse, *cache.args, cache.weights, new_lens=n, last_rows=last)
    assert torch.equal(first.nan_to_num(7.0), cache.weights.nan_to_num(7.0))
    # the slots without keys are still NaN
    assert int(first.isnan().sum()) == first.numel() - Hkv * sum(lens)


def test_rows_that_saw_nothing_and_masked_nan_add_nothing(gpu):
    cache = Cache([90], 2, 16)
    q = queries(cache, 4, 10)
    lse = reference(cache, q, 10, 0)[1].float()[None]
    w = cache.weights.clone()
    lse[0, :, 3] = -math.inf
    ops.fine_key_weights(q, lse, *cache.args, w)
    other = lse.clone()
    other[0, :, 3] = math.inf
    w2 = cache.weights.clone()
    ops.fine_key_weights(q, other, *cache.args, w2)
    assert torch.equal(w.nan_to_num(7.0), w2.nan_to_num(7.0))
    # a key that only the last row sees
    pg, sl = cache.at(0)
    cache.kv[pg[-1], :2, sl[-1]] = float("nan")
    w3 = cache.weights.clone()
    ops.fine_key_weights(q, lse, *cache.args, w3)
    assert torch.equal(w3[pg[:-1], :, sl[:-1]], w[pg[:-1], :, sl[:-1]]) and w3[pg[-1], :, sl[-1]].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,S,page,lens,new,last", [
    (4, 2, 10, 16, [90], None, 0),                                 # one tile of 10 rows, masked and not
    (8, 2, 200, 16, [700, 200], [200, 150], 0),
    (2, 1, 300, 16, [300], None, 100),
    (8, 8, 640, 32, [2000] * 8, None, 0),                          # workgroups of four waves, several ranges
])
def test_rows_taken_out_of_an_account_add_nothing_whatever_they_scored(gpu, Hq, Hkv, S, page, lens, new, last, dtype):
    """LSE = -inf takes a row out: an infinite score of it, or a NaN, leaves the weights as they are without the row."""
    cache, clean = Cache(lens, Hkv, page, dtype), Cache(lens, Hkv, page, dtype)
    q = queries(cache, Hq, S)
    n = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
    out = torch.arange(S) % 3 == 1
    # the key at 2 is infinite in one direction: scores of the rows taken out are +inf, the others' -inf
    size = q[..., 0].abs() + 0.5
    q[..., 0] = torch.where(out.cuda(), size, -size)
    for b in range(len(lens)):
        pg, sl = cache.at(b)
        cache.kv[pg[2], :Hkv, sl[2]] = 0
        cache.kv[pg[2], :Hkv, sl[2], 0] = math.inf
    _, lse = ops.fine_fmha_paged_with_lse(q, *clean.args, new_lens=n)
    lse[:, :, out] = -math.inf
    before, w, want = cache.weights.clone(), cache.weights.clone(), cache.weights.clone()
    ops.fine_key_weights(q, lse, *cache.args, w, new_lens=n, last_rows=last)
    ops.fine_key_weights(q, lse, *clean.args, want, new_lens=n, last_rows=last)
    for b in range(len(lens)):
        pg, sl = cache.at(b)
        want[pg[2], :, sl[2]] = before[pg[2], :, sl[2]]            # (the other rows' probability of that key is nothing)
    assert torch.equal(w.nan_to_num(7.0), want.nan_to_num(7.0))
    for b in range(len(lens)):
        pg, sl = cache.at(b)
        cache.kv[pg[0], :Hkv, sl[0]] = math.nan
        cache.kv[pg[-1], :Hkv, sl[-1]] = -math.inf
    lse.fill_(-math.inf)
    w = before.clone()
    ops.fine_key_weights(q, lse, *cache.args, w, new_lens=n, last_rows=last)
    assert torch.equal(w.nan_to_num(7.0), before.nan_to_num(7.0))


# ---- eviction ------------------------------------------------------------------------------------------------------------


def evicted(cache, budget, recent):
    """What eviction leaves, by plain loops: lengths, pages, weights, positions."""
    kv, w, pos = cache.kv.clone(), cache.weights.clone(), cache.positions.clone()
    lens = []
    for b, n in enumerate(cache.seq_lens):
        lens.append(min(n, budget))
        if n <= budget:
            continue
        pg, sl = (t.tolist() for t in cache.at(b))
        gpg, gsl = cache.at(b)
        for h in range(cache.Hkv):
            wl, pl = cache.weights[gpg, h, gsl].tolist(), cache.positions[gpg, h, gsl].tolist()
            newest = max(pl)

            def rank(j):
                if pl[j] > newest - recent:
                    return (0, 0.0, j)
                return (1, -wl[j], j) if wl[j] == wl[j] else (2, 0.0, j)
            kept = set(sorted(range(n), key=rank)[:budget])
            holes, moved = [j for j in range(budget) if j not in kept], [j for j in range(budget, n) if j in kept]
            assert len(holes) == len(moved)
            d, s = torch.tensor(holes, dtype=torch.long, device="cuda"), torch.tensor(moved, dtype=torch.long, device="cuda")
            for t, i in ((kv, h), (kv, h + cache.Hkv), (w, h), (pos, h)):
                t[gpg[d], i, gsl[d]] = t[gpg[s], i, gsl[s]]
    return lens, kv, w, pos


def positions_of(cache, seed, spread=100):
    gen = torch.Generator().manual_seed(seed)
    for b, n in enumerate(cache.seq_lens):
        pg, sl = cache.at(b)
        cache.positions[pg, :, sl] = torch.stack([torch.randperm(n + spread, generator=gen)[:n] for _ in range(cache.Hkv)], 1).int().cuda()


@pytest.mark.parametrize("kind", ["any", "ties", "equal", "extremes"])
@pytest.mark.parametrize("lens,budget,recent,page,Hkv", [
    ([300], 299, 10, 16, 2), ([64, 65, 63, 0, 200], 64, 64, 16, 2), ([2176, 2048], 2048, 1024, 32, 4), ([1000, 17], 1, 1, 48, 1),
    ([5000, 333], 1001, 0, 16, 2), ([130], 20, 500, 128, 1), ([1], 5, 2, 16, 2), ([40000, 1025], 2049, 64, 64, 1), ([100], 2 ** 31 - 1, 2 ** 31 - 1, 16, 1),
])
def test_eviction(gpu, lens, budget, recent, page, Hkv, kind):
    cache = Cache(lens, Hkv, page, torch.bfloat16, seed=len(lens))
    positions_of(cache, 7)
    gen = torch.Generator().manual_seed(9)
    if kind != "any":
        for b, n in enumerate(lens):
            pg, sl = cache.at(b)
            if kind == "ties":
                x = torch.randint(0, 4, (n, Hkv), generator=gen).float() / 3
            elif kind == "equal":
                x = torch.zeros(n, Hkv)
            else:
                pool = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0, -1.0, 1.1754944e-38])
                x = pool[torch.randint(0, len(pool), (n, Hkv), generator=gen)]
            cache.weights[pg, :, sl] = x.cuda()
    want = evicted(cache, budget, recent)
    lens_before = cache.lens.clone()
    got = ops.fine_evict_paged(*cache.args, cache.weights, cache.positions, budget, recent)
    assert got.tolist() == want[0] and got.dtype == torch.int32 and torch.equal(cache.lens, lens_before)
    for x, y in zip((cache.kv, cache.weights, cache.positions), want[1:]):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("outliers", [False, True], ids=["", "outliers"])
@pytest.mark.parametrize("steps", [1, 40, 3000, 1 << 20])
def test_eviction_of_weights_side_by_side(gpu, steps, outliers):
    """All within `steps` neighbouring values of 32 bits, so that the border is among many that share their upper bits, and with infinities
    and zeros so that those are few of the range's."""
    lens, Hkv = [3000, 700, 9000], 2
    for budget, recent in ((600, 0), (2900, 300), (1, 0)):
        cache = Cache(lens, Hkv, 16, seed=3)
        positions_of(cache, 5)
        gen = torch.Generator().manual_seed(steps)
        for b, n in enumerate(lens):
            pg, sl = cache.at(b)
            w = (0x3f5a0000 + torch.randint(0, steps, (n, Hkv), generator=gen, dtype=torch.int32)).view(torch.float32)
            if outliers:
                w[torch.randperm(n, generator=gen)[:5], 0] = torch.tensor([math.inf, -math.inf, 0.0, -3.0, float("nan")])
                w[:7, 1] = 0.0
            cache.weights[pg, :, sl] = w.cuda()
        want = evicted(cache, budget, recent)
        got = ops.fine_evict_paged(*cache.args, cache.weights, cache.positions, budget, recent)
        assert got.tolist() == want[0]
        for x, y in zip((cache.kv, cache.weights, cache.positions), want[1:]):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("lens,budget,page,Hkv", [([300, 77], 130, 16, 2), ([5000], 2100, 32, 1), ([40000], 9000, 64, 1), ([90, 200], 33, 48, 2)])
def test_eviction_moves_nothing_into_pages_outside_the_pool(gpu, lens, budget, page, Hkv):
    """A slot of such a page holds no key: in front of the budget it stays as it is and so many keys fewer are kept, behind it there is nothing to keep."""
    cache = Cache(lens, Hkv, page)
    positions_of(cache, 3)
    full = cache.table.clone()
    for b, n in enumerate(lens):
        pages = -(-n // page)
        for i in {0, 2 % pages, pages - 1, pages // 2}:
            cache.table[b, i] = (-1, cache.kv.shape[0], 2 ** 31 - 1)[i % 3]
    recent = 10
    kv, w, pos = cache.kv.clone(), cache.weights.clone(), cache.positions.clone()
    there = [torch.tensor([0 <= int(x) < cache.kv.shape[0] for x in row]) for row in cache.table.tolist()]
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        has = [bool(there[b][j // page]) for j in range(n)]
        room = sum(has[:budget])
        pg, sl = full[b].cpu().long()[torch.arange(n) // page].cuda(), (torch.arange(n) % page).cuda()
        for h in range(Hkv):
            wl, pl = cache.weights[pg, h, sl].tolist(), cache.positions[pg, h, sl].tolist()
            newest = max((p for p, x in zip(pl, has) if x), default=0)
            kept = set(sorted((j for j in range(n) if has[j]), key=lambda j: (0, 0.0, j) if pl[j] > newest - recent else (1, -wl[j], j))[:room])
            holes, moved = [j for j in range(budget) if has[j] and j not in kept], [j for j in range(budget, n) if j in kept]
            assert len(holes) == len(moved)
            d, s = torch.tensor(holes, dtype=torch.long, device="cuda"), torch.tensor(moved, dtype=torch.long, device="cuda")
            for t, i in ((kv, h), (kv, h + Hkv), (w, h), (pos, h)):
                t[pg[d], i, sl[d]] = t[pg[s], i, sl[s]]
    got = ops.fine_evict_paged(*cache.args, cache.weights, cache.positions, budget, recent)
    assert got.tolist() == [min(n, budget) for n in lens]
    for x, y in ((cache.kv, kv), (cache.weights, w), (cache.positions, pos)):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("lens,max_pages,budget,recent,kind", [
    ([32768, 20001], 512, 16384, 0, "rising"),        # all 32 keys of a thread, 16384 holes and as many movers
    ([32767, 16387], 512, 5001, 64, "ties"),
    ([30002, 300, 5000], 512, 257, 100, "any"),       # short sequences in a wide table: fewer keys a thread
    ([16385], 257, 16384, 0, "rising"),               # the narrowest table of this kernel
])
def test_eviction_of_sixteen_to_thirty_two_thousand_keys(gpu, lens, max_pages, budget, recent, kind):
    page, Hkv = 64, 2
    cache = Cache(lens, Hkv, page, torch.bfloat16, max_pages=max_pages)
    positions_of(cache, 11)
    gen = torch.Generator().manual_seed(12)
    for b, n in enumerate(lens):
        pg, sl = cache.at(b)
        if kind == "rising":
            cache.weights[pg, :, sl] = torch.arange(n, device="cuda", dtype=torch.float32)[:, None].expand(n, Hkv)
        elif kind == "ties":
            cache.weights[pg, :, sl] = (torch.randint(0, 3, (n, Hkv), generator=gen).float() / 2).cuda()
    want = evicted(cache, budget, recent)
    got = ops.fine_evict_paged(*cache.args, cache.weights, cache.positions, budget, recent)
    assert got.tolist() == want[0]
    for x, y in zip((cache.kv, cache.weights, cache.positions), want[1:]):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def test_eviction_with_positions_of_the_whole_range(gpu):
    cache = Cache([100], 1, 16)
    pg, sl = cache.at(0)
    cache.positions[pg, 0, sl] = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, -1] * 25, dtype=torch.int32, device="cuda")
    for recent in (0, 1, 2 ** 31 - 1):
        want = evicted(cache, 40, recent)
        c2 = [cache.kv.clone(), cache.weights.clone(), cache.positions.clone()]
        ops.fine_evict_paged(c2[0], cache.table, cache.lens, c2[1], c2[2], 40, recent)
        for x, y in zip(c2, want[1:]):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


# ---- streams, graphs, a loop of all of them ---------------------------------------------------------------------------------


class Loop:
    """A generation loop over one cache: prompts are filed, what they attended to is counted, then steps with eviction."""

    def __init__(self, seed=0, dtype=torch.float16):
        gen = torch.Generator().manual_seed(seed)
        self.Hq, self.Hkv, self.page, self.budget, self.recent = 8, 2, 16, 90, 30
        self.prompts = [120, 33, 77]
        self.cache = Cache([0, 0, 0], self.Hkv, self.page, dtype, spare=40, max_pages=9)
        perm = torch.randperm(40, generator=gen)[:27].int().reshape(3, 9)
        self.cache.table.copy_(perm)
        angle = torch.arange(400, dtype=torch.double)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.double) / 64)
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        self.prompt = torch.randn(3, 120, self.Hq + 2 * self.Hkv, D, generator=gen).to(dtype).cuda()
        self.tokens = torch.randn(12, 3, 1, self.Hq + 2 * self.Hkv, D, generator=gen).to(dtype).cuda()
        self.next = torch.tensor(self.prompts, dtype=torch.int32, device="cuda")   # position of the next token

    def prefill(self):
        c, new = self.cache, torch.tensor(self.prompts, dtype=torch.int32, device="cuda")
        c.lens.copy_(new)
        qkv = self.prompt.clone()
        ops.fine_rope_paged(qkv, *c.args, self.cos, self.sin, torch.arange(120, dtype=torch.int32, device="cuda"), self.Hq, new_lens=new, weights=c.weights,
                            key_positions=c.positions, keep_keys=True)
        q, k, v = (t.transpose(1, 2) for t in qkv.split((self.Hq, self.Hkv, self.Hkv), 2))
        o, lse = ops.fine_fmha_with_lse(q, k, v, True)
        paged, lse2 = ops.fine_fmha_paged_with_lse(q, *c.args, new_lens=new)
        ops.fine_key_weights(q, lse, *c.args, c.weights, new_lens=new)
        return q, o, lse, paged, lse2

    def step(self, qkv):
        c = self.cache
        c.lens.add_(1)
        ops.fine_rope_paged(qkv, *c.args, self.cos, self.sin, self.next[:, None].contiguous(), self.Hq, weights=c.weights, key_positions=c.positions)
        q = qkv[:, :, :self.Hq].transpose(1, 2)
        o, lse = ops.fine_fmha_paged_with_lse(q, *c.args, weights=c.weights)
        c.lens.copy_(ops.fine_evict_paged(*c.args, c.weights, c.positions, self.budget, self.recent))
        self.next.add_(1)
        return q, o, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_a_generation_loop(gpu, dtype):
    loop = Loop(dtype=dtype)
    c = loop.cache
    q, o, lse, paged, lse2 = loop.prefill()
    c.seq_lens = list(loop.prompts)
    for b, n in enumerate(loop.prompts):
        # the prompt's attention over its own projection and over the pages are the same sums, each within its rounding (half a step of the
        # probabilities and of the result, values up to 5)
        assert (o[b, :, :n].double() - paged[b, :, :n].double()).abs().max() <= 4 * HALF_STEP[dtype] * 5
        # the prompt's kernel sums the probabilities as rounded for the second product (`l[qb] += 1 P^T` in csrc/fmha_fwd.hip): each is off
        # by at most half a step h of its value, so the sum by a factor within 1 +- h and its logarithm by at most h + h^2
        h = HALF_STEP[dtype]
        assert (lse[b, :, :n] - lse2[b, :, :n]).abs().max() <= h + h * h + 1e-5
        assert (paged[b, :, n:] == 0).all()
    check_attention(c, q, paged, lse2, loop.prompts)
    for b, n in enumerate(loop.prompts):
        pg, sl = c.at(b)
        # every row's probabilities sum to one, as far as its log-sum-exp goes (above)
        assert (c.weights[pg, :, sl].double().sum(0) - n * 4).abs().max() <= n * 4 * (h + h * h + 1e-5)
        assert (c.positions[pg, :, sl] == torch.arange(n, device="cuda")[:, None]).all()
    for i in range(12):
        c.lens.copy_(torch.tensor(c.seq_lens, dtype=torch.int32))
        # what the step must leave is worked out between its calls
        c.seq_lens = [n + 1 for n in c.seq_lens]
        qkv = loop.tokens[i].clone()
        c.lens.add_(1)
        ops.fine_rope_paged(qkv, *c.args, loop.cos, loop.sin, loop.next[:, None].contiguous(), loop.Hq, weights=c.weights, key_positions=c.positions)
        before = c.weights.clone()
        q = qkv[:, :, :loop.Hq].transpose(1, 2)
        o, lse = ops.fine_fmha_paged_with_lse(q, *c.args, weights=c.weights)
        check_attention(c, q, o, lse, None, before)
        want = evicted(c, loop.budget, loop.recent)
        lens = ops.fine_evict_paged(*c.args, c.weights, c.positions, loop.budget, loop.recent)
        assert lens.tolist() == want[0]
        for x, y in zip((c.kv, c.weights, c.positions), want[1:]):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
        c.seq_lens = want[0]
        loop.next.add_(1)


def state_of(loop):
    c = loop.cache
    return [t.clone() for t in (c.kv, c.weights, c.positions, c.lens, loop.next)]


def test_a_captured_step_is_replayed_as_the_lengths_go_on(gpu):
    eager, graph = Loop(), Loop()
    eager.prefill()
    graph.prefill()
    token = graph.tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = state_of(graph)
    with torch.cuda.stream(side):
        graph.step(token)                       # once before the capture
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = graph.step(token)
    c = graph.cache
    for t, s in zip((c.kv, c.weights, c.positions, c.lens, graph.next), saved):
        t.copy_(s)
    for i in range(12):
        token.copy_(graph.tokens[i])
        g.replay()
        want = eager.step(eager.tokens[i].clone())
        torch.cuda.synchronize()
        assert torch.equal(out[1], want[1]) and torch.equal(out[2], want[2])
        for x, y in zip(state_of(graph), state_of(eager)):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("Hq,Hkv,S", [(1, 1, 1), (4, 2, 1), (32, 8, 1), (64, 8, 1), (16, 2, 4), (40, 4, 7)])
def test_captured_and_eager_calls_give_the_same_bits(gpu, Hq, Hkv, S):
    """Long caches are cut into parts, joined in an order that the lengths alone decide."""
    cache = Cache([9000, 17, 0, 3000], Hkv, 32)
    q = queries(cache, Hq, S)
    weights = cache.weights.clone()
    eager = [ops.fine_fmha_paged_with_lse(q, *cache.args, weights=weights) for _ in range(3)]
    check_attention(cache, q, *eager[0])
    for o, lse in eager[1:]:
        assert torch.equal(o, eager[0][0]) and torch.equal(lse, eager[0][1])
    other = cache.weights.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.fine_fmha_paged_with_lse(q, *cache.args, weights=other)
    for _ in range(3):
        g.replay()
        again = ops.fine_fmha_paged(q, *cache.args)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0][0]) and torch.equal(out[1], eager[0][1]) and torch.equal(again, out[0])
    assert torch.equal(other.nan_to_num(7.0), weights.nan_to_num(7.0))


def test_calls_on_two_streams_at_once(gpu):
    loops = [Loop(seed=s) for s in (1, 2)]
    alone = [Loop(seed=s) for s in (1, 2)]
    results = []
    for loop in alone:
        loop.prefill()
        results.append([loop.step(t.clone()) for t in loop.tokens])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in loops]
    got = [[], []]
    for s, loop in zip(streams, loops):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            loop.prefill()
    for i in range(12):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(loops[k].step(loops[k].tokens[i].clone()))
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in zip(got[k], results[k]):
            assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
        for x, y in zip(state_of(loops[k]), state_of(alone[k])):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def test_strides_that_mean_nothing_and_strides_that_are_too_large(gpu):
    c = Cache([40], 2, 16, spare=0)
    assert c.kv.shape[0] == 3
    q = queries(c, 8, 1)
    want = ops.fine_fmha_paged(q, *c.args)
    # one sequence, one row: their strides may be anything
    odd = torch.empty(8 * D + 5, dtype=torch.float16, device="cuda")[:8 * D].as_strided((1, 8, 1, D), (7, D, 3, 1))
    odd.copy_(q)
    table = c.table.as_strided(c.table.shape, (1, 1))
    assert torch.equal(ops.fine_fmha_paged(odd, c.kv, table, c.lens), want)
    # rows 2^24 elements apart, an unaligned start, a reversed order of dimensions
    S = 3
    q = queries(c, 8, S)
    want, lse = ops.fine_fmha_paged_with_lse(q, *c.args)
    w = [c.weights.clone() for _ in range(4)]
    ops.fine_key_weights(q, lse, *c.args, w[0])
    far = torch.empty((S - 1) * (1 << 24) + 8 * D, dtype=torch.float16, device="cuda").as_strided((1, 8, S, D), (8, D, 1 << 24, 1))
    shifted = torch.empty(8 * S * D + 1, dtype=torch.float16, device="cuda")[1:].view(1, 8, S, D)
    across = torch.empty(D, S, 8, 1, dtype=torch.float16, device="cuda").permute(3, 2, 1, 0)
    for i, other in enumerate((far, shifted, across)):
        other.copy_(q)
        assert torch.equal(ops.fine_fmha_paged(other, *c.args), want)
        ops.fine_key_weights(other, lse, *c.args, w[i + 1])
        assert torch.equal(w[i + 1].nan_to_num(7.0), w[0].nan_to_num(7.0))
    # a pool of one page
    one = Cache([10], 2, 16, spare=0)
    pool = one.kv.as_strided(one.kv.shape, (3,) + one.kv.stride()[1:])
    q = queries(one, 8, 1)
    assert torch.equal(ops.fine_fmha_paged(q, pool, one.table, one.lens), ops.fine_fmha_paged(q, *one.args))


def test_as_many_sequences_as_a_call_takes(gpu):
    """65528 (sequence, kv head) pairs: a call gives what calls of parts of the batch give."""
    B, Hkv, page, P = 8191, 8, 16, 40
    gen = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn((B * P, 2 * Hkv, page, D), generator=gen, device="cuda", dtype=torch.float16)
    table = torch.randperm(B * P, generator=gen, device="cuda").int().reshape(B, P)
    lens = torch.randint(0, P * page + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    weights = torch.rand((B * P, Hkv, page), generator=gen, device="cuda")
    positions = torch.randint(0, 5000, (B * P, Hkv, page), generator=gen, device="cuda", dtype=torch.int32)
    parts = [slice(0, 3000), slice(3000, 8000), slice(8000, B)]
    for S in (1, 40):                                              # one token; a chunk, whose account is worked out from the log-sum-exp
        q = torch.randn((B, Hkv, S, D), generator=gen, device="cuda", dtype=torch.float16)
        a, b = weights.clone(), weights.clone()
        o, lse = ops.fine_fmha_paged_with_lse(q, kv, table, lens, weights=a)
        for p in parts:
            po, pl = ops.fine_fmha_paged_with_lse(q[p], kv, table[p], lens[p], weights=b)
            # (a cut at another place: rounding of 16-bit probabilities and results, |v| <= 6, and of the sums)
            assert ((o[p] - po).abs() <= 4 * 2.0 ** -11 * 6).all() and (lse[p] - pl).abs().nan_to_num(0.0).max() <= 1e-5
            assert torch.equal(lse[p].isinf(), pl.isinf())
        # a probability is off by 2^-16 of itself at most in each (a score and its row's log-sum-exp, 2^-17 each), their sum is below b
        assert ((a - b).abs() <= 2 * 2.0 ** -16 * b + 1e-6).all()
    two = [[t.clone() for t in (kv, weights, positions)] for _ in range(2)]
    left = ops.fine_evict_paged(two[0][0], table, lens, two[0][1], two[0][2], 300, 40)
    for p in parts:
        assert torch.equal(left[p], ops.fine_evict_paged(two[1][0], table[p], lens[p], two[1][1], two[1][2], 300, 40))
    assert all(torch.equal(x, y) for x, y in zip(*two)) and torch.equal(left, lens.clamp(max=300))
    qkv = torch.randn((B, 2, 3 * Hkv, D), generator=gen, device="cuda", dtype=torch.float16)
    t, other = torch.rand((5000, 64), generator=gen, device="cuda"), qkv.clone()
    pos = torch.randint(0, 5000, (B, 2), generator=gen, device="cuda", dtype=torch.int32)
    ops.fine_rope_paged(qkv, two[0][0], table, left, t, t, pos, Hkv, weights=two[0][1], key_positions=two[0][2])
    for p in parts:
        ops.fine_rope_paged(other[p], two[1][0], table[p], left[p], t, t, pos[p], Hkv, weights=two[1][1], key_positions=two[1][2])
    assert torch.equal(qkv, other) and all(torch.equal(x, y) for x, y in zip(*two))


def test_sequences_may_share_pages_that_are_only_read(gpu):
    """A common beginning of two texts in the same pages, and a page that a sequence has twice."""
    cache = Cache([320, 200, 97], 2, 16)
    cache.table[1, :6] = cache.table[0, :6]
    cache.table[2, 3] = cache.table[2, 1]
    for S in (1, 40):
        q = queries(cache, 8, S)
        check_attention(cache, q, *ops.fine_fmha_paged_with_lse(q, *cache.args))


def test_operators_through_the_dispatcher_are_the_same(gpu):
    cache = Cache([700, 31], 2, 16)
    q = queries(cache, 8, 2)
    direct, lse = ops.fine_fmha_paged_with_lse(q, *cache.args)
    through = torch.ops.fmha_unified
    assert torch.equal(through.finefmha_paged(q, *cache.args, None, None), direct)
    o, l = through.finefmha_paged_lse(q, *cache.args, None, None)
    assert torch.equal(o, direct) and torch.equal(l, lse)
    w = [cache.weights.clone(), cache.weights.clone()]
    ops.fine_key_weights(q, lse, *cache.args, w[0])
    through.key_weights(q, lse, *cache.args, w[1], None, 0)
    assert torch.equal(w[0].nan_to_num(7.0), w[1].nan_to_num(7.0))
    positions_of(cache, 1)
    a = [t.clone() for t in (cache.kv, cache.weights, cache.positions)]
    b = [t.clone() for t in a]
    assert torch.equal(ops.fine_evict_paged(a[0], cache.table, cache.lens, a[1], a[2], 20, 5),
                       through.evict_paged(b[0], cache.table, cache.lens, b[1], b[2], 20, 5))
    assert all(torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)) for x, y in zip(a, b))
    qkv = torch.randn(2, 3, 12, D, device="cuda").half()
    t, pos = torch.rand(50, 64, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    x, y = qkv.clone(), qkv.clone()
    ops.fine_rope_paged(x, a[0], cache.table, cache.lens, t, t, pos, 8)
    through.rope_paged(y, b[0], cache.table, cache.lens, t, t, pos, 8, None, None, None, False)
    assert torch.equal(x, y) and torch.equal(a[0].nan_to_num(7.0), b[0].nan_to_num(7.0))


def test_gradients_that_there_are_none_of_are_not_lost_in_silence(gpu):
    """As with the operators that go through torch's dispatcher: the result of a tensor that needs a gradient needs one, and going back through it is not silent."""
    cache = Cache([70, 31], 2, 16)
    q = queries(cache, 8, 2)
    want = ops.fine_fmha_paged(q, *cache.args)
    k = torch.zeros(2, 2, 70, D, dtype=torch.float16, device="cuda")
    other = q.clone().requires_grad_()
    expected, _ = ops.fine_fmha_with_lse(other, k, k, True)
    o = ops.fine_fmha_paged(other, *cache.args)
    o2, lse = ops.fine_fmha_paged_with_lse(other, *cache.args)
    assert o.requires_grad == o2.requires_grad == lse.requires_grad == expected.requires_grad
    assert torch.equal(o, want) and torch.equal(o2, want)
    with torch.no_grad():
        assert not ops.fine_fmha_paged(other, *cache.args).requires_grad
    # (torch has no way of its own to batch an operator that may write an argument, and says so)
    with pytest.raises(RuntimeError, match="Batching rule not implemented for fmha_unified::finefmha_paged"):
        torch.vmap(lambda x: ops.fine_fmha_paged(x, *cache.args))(torch.stack((q, -q)))


def test_operators_refuse_wrong_tensors_on_the_gpu(gpu):
    c = Cache([40, 20], 2, 16)
    q = queries(c, 8, 1)
    one = torch.ones(50, 64, device="cuda")
    pos = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(2, 1, 12, D, dtype=torch.float16, device="cuda")
    lse = torch.zeros(2, 8, 1, device="cuda")

    def refused(match, f, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)

    refused("q must be", ops.fine_fmha_paged, q[:1], *c.args)
    refused("q must be", ops.fine_fmha_paged, q.bfloat16(), *c.args)
    refused("multiple of Hkv", ops.fine_fmha_paged, q[:, :7], *c.args)
    refused("block_table", ops.fine_fmha_paged, q, c.kv, c.table.long(), c.lens)
    refused("block_table", ops.fine_fmha_paged, q, c.kv, c.table.cpu(), c.lens)
    refused("seq_lens", ops.fine_fmha_paged, q, c.kv, c.table, c.lens[:1])
    refused("new_lens", ops.fine_fmha_paged, q, *c.args, new_lens=c.lens.long())
    refused("weights", ops.fine_fmha_paged, q, *c.args, weights=c.weights.half())
    refused("weights", ops.fine_fmha_paged, q, *c.args, weights=c.weights[:, :1])
    refused("page_size", ops.fine_fmha_paged, q, c.kv[:, :, :15], c.table, c.lens)
    refused("qkv must be", ops.fine_rope_paged, qkv, *c.args, one, one, pos, 7)
    refused("cos and sin", ops.fine_rope_paged, qkv, *c.args, one, one.half(), pos, 8)
    refused("positions", ops.fine_rope_paged, qkv, *c.args, one, one, pos[:1], 8)
    refused("key_positions", ops.fine_rope_paged, qkv, *c.args, one, one, pos, 8, key_positions=c.weights)
    refused("lse", ops.fine_key_weights, q, lse[:, :4], *c.args, c.weights)
    refused("last_rows", ops.fine_key_weights, q, lse, *c.args, c.weights, last_rows=-1)
    refused("budget", ops.fine_evict_paged, *c.args, c.weights, c.positions, 0, 1)
    refused("key_positions", ops.fine_evict_paged, *c.args, c.weights, c.positions.float(), 5, 1)
