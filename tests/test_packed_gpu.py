"""Packed batches against plain loops in 64 bits: plans from lengths, filing by slots, attention of whole prompts."""
import math
import random

import pytest
import torch

import fmha_unified
import mi355_serving as lib
from reference64 import D, HALF_STEP, attention64, check

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets_of(lens):
    return ints([sum(lens[:b]) for b in range(len(lens) + 1)])


# ---- attention of whole prompts ----------------------------------------------------------------------------------------


def batch(lens, Hq, Hkv, dtype, spare=0, seed=0, layout="fused", scale=1.5):
    """q, k, v of a batch whose rows behind the last sequence are NaN."""
    gen = torch.Generator().manual_seed(seed)
    rows, heads = sum(lens) + spare, Hq + 2 * Hkv
    x = torch.randn(rows, heads, D, generator=gen)
    x[:, :Hq] *= scale
    x[sum(lens):] = math.nan
    x = x.to(dtype).cuda()
    if layout == "heads":        # head-major
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "odd":          # an address and strides that no kernel reads in place
        y = torch.empty(rows * heads * (D + 1) + 1, dtype=dtype, device="cuda")[1:].view(rows, heads, D + 1)[..., :D]
        y.copy_(x)
        x = y
    parts = x.split((Hq, Hkv, Hkv), 1)
    return [p.contiguous() for p in parts] if layout == "apart" else parts


def check_packed(q, k, v, lens, o, lse, causal=True, first=0):
    at = first
    for n in lens:
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril()
        rows = slice(at, at + n)
        if n:
            check(o[rows].transpose(0, 1), lse[:, rows], attention64(q[rows].transpose(0, 1), k[rows].transpose(0, 1), v[rows].transpose(0, 1), seen))
        at += n
    for rows in (slice(0, first), slice(at, None)):
        assert (o[rows] == 0).all() and (lse[:, rows] == -math.inf).all()


PACKED = [   # Hq, Hkv, lengths, options
    (8, 2, [1], {}),
    (8, 2, [77, 5, 1], {}),
    (32, 8, [129, 0, 128, 127, 0, 64, 63, 65, 2], dict(spare=3)),
    (32, 8, [300, 257, 1, 256, 255], dict(layout="apart", spare=130)),
    (16, 4, [1000, 17], dict(layout="heads")),
    (8, 8, [513, 40], dict(layout="odd", spare=1)),
    (64, 8, [700], dict(spare=1)),
    (40, 8, [64, 640], {}),
    (1, 1, [2049], {}),
    (6, 3, [191, 193, 192], {}),
    (4, 1, [(37 * i) % 41 for i in range(70)], dict(spare=7)),            # more than 64 sequences
    (2, 1, [(7 * i) % 5 for i in range(2500)], dict(spare=70)),           # more than 1024
    (32, 8, [0, 0, 0], dict(spare=5)),
    (16, 1, [100, 33, 5], {}),                                             # more heads a kv head than lie side by side
    (8, 1, [(53 * i) % 150 for i in range(64)], dict(spare=1)),           # as many sequences as a workgroup orders
    (12, 4, [(53 * i) % 150 for i in range(65)], {}),
    (32, 8, [256] * 16, {}),                                               # as many items for every workgroup
    (16, 16, [2000, 30, 700, 1], {}),                                      # few and long ones, workgroups of which have one more than others
    (24, 8, [(71 * i) % 400 for i in range(40)], {}),
    (16, 8, [1100, 900, 1300], {}),
]


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("case", PACKED, ids=lambda c: "%d-%d-B%d-%s-%s" % (c[0], c[1], len(c[2]), sum(c[2]), c[3].get("layout", "fused")))
def test_attention_of_prompts(gpu, case, causal, dtype):
    Hq, Hkv, lens, options = case
    q, k, v = batch(lens, Hq, Hkv, dtype, **options)
    o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of(lens), causal)
    assert o.is_contiguous() and o.shape == q.shape and o.dtype == dtype and lse.shape == (Hq, q.shape[0]) and lse.dtype == torch.float32
    check_packed(q, k, v, lens, o, lse, causal)
    again, lse2 = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of(lens), causal)
    assert torch.equal(o, again) and torch.equal(lse, lse2)
    assert torch.equal(o, ops.fine_fmha_packed(q, k, v, offsets_of(lens), causal))


def pinned(q, k, v, offsets, causal, variant):
    cdll, (rows, Hq, _), Hkv = lib.load(), q.shape, k.shape[1]
    o, lse = torch.empty(q.shape, dtype=q.dtype, device="cuda"), torch.empty(Hq, rows, device="cuda")
    need = cdll.mi355_fmha_packed_workspace_bytes(rows, len(offsets) - 1, Hq, Hkv)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    import ctypes
    st = (ctypes.c_int64 * 8)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), o.stride(0), o.stride(1))
    rc = cdll.mi355_internal_fmha_packed_variant(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), offsets.data_ptr(), rows, len(offsets) - 1, Hq, Hkv,
                                                 st, D ** -0.5, int(causal), int(q.dtype == torch.bfloat16), ws.data_ptr(), need, variant, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, cdll.mi355_last_error()
    return o, lse


@TYPES
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("case", [(8, 2, [300, 1, 700]), (16, 8, [513, 129, 64, 33]), (32, 8, [257] * 9 + [1]), (64, 8, [40, 1600])], ids=lambda c: "%d-%d-%d" % (c[0], c[1], sum(c[2])))
def test_both_sizes_of_q_tiles(gpu, case, variant, dtype):
    Hq, Hkv, lens = case
    q, k, v = batch(lens, Hq, Hkv, dtype, spare=2)
    for causal in (True, False):
        check_packed(q, k, v, lens, *pinned(q, k, v, offsets_of(lens), causal, variant), causal)


@TYPES
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("where", ["values", "keys", "queries"])
def test_what_a_row_does_not_see_has_no_influence(gpu, where, variant, dtype):
    """Infinities and NaN in the rows behind a row, in its sequence and in the others; the rows that see them come out as the formula has it."""
    lens = [70, 300, 513, 9]
    q, k, v = batch(lens, 8, 2, dtype, spare=4, scale=0.2)
    at = {0: (69, math.nan), 1: (70 + 200, math.inf), 2: (370 + 255, math.nan), 3: (370 + 512, -math.inf)}
    x = dict(values=v, keys=k, queries=q)[where]
    for row, value in at.values():
        x[row, 1, 5] = value
    o, lse = pinned(q, k, v, offsets_of(lens), True, variant)
    if where == "keys":   # (a score that is infinite: the formula gives NaN, or leaves the key out; which rows they reach is what counts here)
        first = 0
        for n in lens:
            bad = [row - first for row, _ in at.values() if first <= row < first + n]
            good = slice(first, first + (min(bad) if bad else n))
            seen = torch.ones(good.stop - first, good.stop - first, dtype=torch.bool, device="cuda").tril()
            check(o[good].transpose(0, 1), lse[:, good], attention64(q[good].transpose(0, 1), k[good].transpose(0, 1), v[good].transpose(0, 1), seen))
            first += n
        return
    if where == "queries":
        for row, _ in at.values():
            assert o[row, 1].isnan().all() and not o[row, 0].isnan().any()
            q[row, 1] = o[row, 1] = 0
            lse[1, row] = 0
        keep = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
        keep[[row for row, _ in at.values()]] = False
        want_o, want_lse = pinned(q, k, v, offsets_of(lens), True, variant)
        assert torch.equal(o[keep], want_o[keep]) and torch.equal(lse[:, keep], want_lse[:, keep])
        return
    check_packed(q, k, v, lens, o, lse)


def test_a_whole_batch_of_nan_ends(gpu):
    q, k, v = batch([3000, 3000], 8, 2, torch.float16)
    for x in (q, k, v):
        x.fill_(math.nan)
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of([3000, 3000]))
        assert o.isnan().all() and lse.isnan().all()


def test_offsets_that_are_wrong_leave_the_rest_alone(gpu):
    q, k, v = batch([200, 100], 8, 2, torch.float16)
    for offsets, lens, first in (([0, 200, 100, 300], [200, 0, 100], 0), ([0, 200, 100], [200], 0), ([0, 200, 100, 250, 20], [200, 0, 50], 0), ([0, 200, 900], [200, 100], 0), ([-5, 200, 300], [200, 100], 0), ([50, 100, 120], [50, 20], 50), ([400, 500], [0], 300)):
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, ints(offsets))
        check_packed(q, k, v, lens, o, lse, first=first)


def test_scores_of_every_size(gpu):
    """Rows of one key, of equal scores, and of scores so far apart that one key has it all."""
    for scale in (1e-4, 1.0, 40.0):
        q, k, v = batch([1, 130, 300], 8, 2, torch.bfloat16, scale=scale)
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of([1, 130, 300]))
        if scale < 40:
            check_packed(q, k, v, [1, 130, 300], o, lse)
        else:
            assert o.isfinite().all() and lse.isfinite().all() and (o[0] == v[0].repeat_interleave(4, 0)).all()


@pytest.mark.parametrize("Hq, lens, variant", [(4, [8191, 100], 0), (8, [8192], 1), (8, [5, 8191, 0, 100], 1)], ids=["8191", "512-tiles", "more-tiles"])
def test_a_long_prompt(gpu, Hq, lens, variant):
    """Tiles of 16 rows of 8 heads: a sequence of as many as a workgroup orders by itself, and a batch that may have more."""
    q, k, v = batch(lens, Hq, 1, torch.bfloat16)
    check_packed(q, k, v, lens, *pinned(q, k, v, offsets_of(lens), True, variant))


def test_more_rows_than_the_list_has_bins_for(gpu):
    lens = [(97 * i) % 500 for i in range(300)]
    q, k, v = batch(lens, 1, 1, torch.float16)
    assert sum(lens) > 64 * 1024
    for causal in (True, False):
        check_packed(q, k, v, lens, *ops.fine_fmha_packed_with_lse(q, k, v, offsets_of(lens), causal), causal)


def test_rows_that_lie_beyond_32_bits(gpu):
    """Rows 2^20 elements apart, 4.4 GB from first to last."""
    rows, lens = 2200, [2000, 200]
    whole = torch.empty(rows << 20, dtype=torch.float16, device="cuda")
    x = torch.as_strided(whole, (rows, 6, D), (1 << 20, D, 1))
    x.copy_(torch.randn(rows, 6, D, generator=torch.Generator().manual_seed(4)).half())
    q, k, v = x.split((4, 1, 1), 1)
    o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of(lens))
    want, want_lse = ops.fine_fmha_packed_with_lse(*(t.contiguous() for t in (q, k, v)), offsets_of(lens))
    assert torch.equal(o, want) and torch.equal(lse, want_lse)
    kv, (cos, sin) = torch.zeros(140, 2, 16, D, dtype=torch.float16, device="cuda"), tables(rows)
    at, other, kv2 = torch.arange(rows, dtype=torch.int32, device="cuda"), x.contiguous(), torch.zeros_like(kv)
    ops.fine_rope_packed(x, kv, at, cos, sin, at, 4)
    ops.fine_rope_packed(other, kv2, at, cos, sin, at, 4)
    assert torch.equal(x, other) and torch.equal(kv, kv2) and (kv != 0).any()


def test_captured_calls_serve_the_lengths_of_their_tensors(gpu):
    q, k, v = batch([900], 16, 4, torch.float16)
    offsets = offsets_of([900, 0, 0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.fine_fmha_packed_with_lse(q, k, v, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets)
        o2, lse2 = ops.fine_fmha_packed_with_lse(q, k, v, offsets, False)
    for lens in ([900, 0, 0], [300, 300, 300], [1, 0, 898], [0, 0, 0], [5, 600, 7]):
        offsets.copy_(offsets_of(lens))
        graph.replay()
        want = ops.fine_fmha_packed_with_lse(q, k, v, offsets)
        want2 = ops.fine_fmha_packed_with_lse(q, k, v, offsets, False)
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and torch.equal(o2, want2[0]) and torch.equal(lse2, want2[1])
        check_packed(q, k, v, lens, o, lse)


def test_two_streams_at_once(gpu):
    a, b = batch([700, 30], 16, 4, torch.float16, seed=1), batch([64] * 20, 16, 4, torch.float16, seed=2)
    want = ops.fine_fmha_packed(*a, offsets_of([700, 30])), ops.fine_fmha_packed(*b, offsets_of([64] * 20))
    oa, ob = offsets_of([700, 30]), offsets_of([64] * 20)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s):
            got.append((ops.fine_fmha_packed(*a, oa), 0))
        with torch.cuda.stream(t):
            got.append((ops.fine_fmha_packed(*b, ob), 1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for x, i in got)


# ---- plans -------------------------------------------------------------------------------------------------------------


class Pool:
    """Lengths, table and ring of a pool, on the host and on the device."""

    def __init__(self, B, columns, n_pages, page, positions=True, seed=0, stride=None):
        self.rng = random.Random(seed)
        order = list(range(n_pages))
        self.rng.shuffle(order)
        self.page, self.n_pages, self.columns = page, n_pages, columns
        self.table, self.lens, self.ring, self.span = [[-1] * columns for _ in range(B)], [0] * B, order, [0, n_pages]
        self.texts = [self.rng.randrange(50) for _ in range(B)] if positions else None
        whole = torch.full((B, stride or columns), -9, dtype=torch.int32, device="cuda")
        self.d_table = whole[:, :columns]
        self.d = None
        self.put()

    def put(self):
        self.d_table.copy_(ints(self.table))
        self.d = [ints(self.lens), ints(self.ring), ints(self.span), ints(self.texts) if self.texts else None]

    def plan(self, new, rows):
        """The same on the host; (offsets, positions, slots, taken)."""
        page, n_pages = self.page, self.n_pages
        first, count = self.span
        free = [self.ring[(first + i) % n_pages] for i in range(count)]
        offsets, positions, slots, taken, back, lacked, used = [0], [-1] * rows, [-1] * rows, [], [], 0, 0
        for b, n in enumerate(max(x, 0) for x in new):
            at, have, row = offsets[-1], self.lens[b], self.table[b]
            offsets.append(min(at + n, rows))
            ok = at + n <= rows and have + n <= self.columns * page
            lacks = [c for c in range(have // page, -(-(have + n) // page)) if not 0 <= row[c] < n_pages] if ok and n else []
            lacked += len(lacks)
            ok = ok and (not lacks or lacked <= count)
            taken.append(n if ok else 0)
            if ok:
                for c in lacks:
                    row[c] = free[used]
                    used += 1
                for t in range(n):
                    positions[at + t] = (self.texts[b] if self.texts else have) + t
                    slots[at + t] = row[(have + t) // page] * page + (have + t) % page
                self.lens[b] += n
                if self.texts:
                    self.texts[b] += n
            for c in range(-(-self.lens[b] // page), self.columns):
                if 0 <= row[c] < n_pages:
                    back.append(row[c])
                    row[c] = -1
        for i, p in enumerate(back):
            self.ring[(first + count + i) % n_pages] = p
        self.span = [(first + used) % n_pages, count - used + len(back)]
        return offsets, positions, slots, taken

    def run(self, new, rows):
        lens, ring, span, texts = self.d
        return ops.fine_plan_packed(self.d_table, lens, new, ring, span, self.page, rows, next_positions=texts)

    def step(self, new, rows):
        got, want = self.run(ints(new), rows), self.plan(new, rows)
        for name, g, w in zip(("offsets", "positions", "slots", "taken"), got, want):
            assert g.dtype == torch.int32 and g.tolist() == w, name
        self.same()
        return got

    def same(self):
        lens, ring, span, texts = self.d
        assert self.d_table.tolist() == self.table and lens.tolist() == self.lens and span.tolist() == self.span
        assert texts is None or texts.tolist() == self.texts
        at, n = self.span
        free = [self.ring[(at + i) % self.n_pages] for i in range(n)]
        r = ring.tolist()
        assert [r[(at + i) % self.n_pages] for i in range(n)] == free
        held = [p for row in self.table for p in row if p >= 0]
        assert sorted(held + free) == list(range(self.n_pages))   # no page is lost or held twice


@pytest.mark.parametrize("shape", [(1, 4, 9, 16), (3, 7, 15, 16), (70, 30, 900, 48), (300, 9, 1500, 32), (5, 700, 1900, 16), (2, 20, 64, 128)], ids=lambda s: "B%d-c%d-n%d-p%d" % s)
@pytest.mark.parametrize("positions", [False, True], ids=["keys", "texts"])
def test_plans_of_a_run_of_requests(gpu, shape, positions):
    """Prompts, steps, drafts that are taken back, sequences that end: rows that do not suffice, tables that are full and pools that run out among them."""
    B, columns, n_pages, page = shape
    pool = Pool(B, columns, n_pages, page, positions, stride=columns + 3)
    rng, seen = random.Random(B * columns), set()
    most = columns * page
    for step in range(25):
        new = []
        for b in range(B):
            kind = rng.random()
            if kind < 0.15 and pool.lens[b]:
                pool.lens[b] = 0 if kind < 0.08 else rng.randrange(pool.lens[b])   # done, or cut
                new.append(rng.choice((0, 1, -3)))
            elif kind < 0.3:
                new.append(rng.randrange(1, max(2, int(most * 0.7) if pool.lens[b] == 0 else most // 4)))
            else:
                new.append(rng.choice((0, 1, 1, 1, 5, page)))
        pool.d[0].copy_(ints(pool.lens))
        total = sum(max(x, 0) for x in new)
        rows = max(0, total + rng.choice((0, 0, 1, 77, 5000, -3, -total // 2)))
        taken = pool.step(new, rows)[3].tolist()
        seen.update(("short" if t < n else "taken") for t, n in zip(taken, new) if n > 0)
    assert seen == {"short", "taken"}


def test_a_plan_of_no_rows_gives_pages_back(gpu):
    pool = Pool(3, 5, 12, 16)
    pool.step([50, 20, 30], 100)
    pool.lens = [17, 0, 30]
    pool.d[0].copy_(ints(pool.lens))
    offsets, positions, slots, taken = pool.step([0, 0, 0], 0)
    assert positions.numel() == slots.numel() == 0 and offsets.tolist() == [0] * 4


def test_lengths_and_spans_out_of_range_stay_inside(gpu):
    """What no program should hand in gives some plan, and no access outside the tensors."""
    table = ints([[0, 1, 99, -5], [2, 2, 2, 2], [7, -1, -1, -1]])
    for lens, new, span in (([-7, 1 << 30, 5], [1 << 30, 3, 20], [-3, 99]), ([64, 0, 17], [-1, 2147483647, 40], [2147483647, -2147483648]), ([0, 0, 0], [16] * 3, [7, 8])):
        guard = torch.full((64,), 77, dtype=torch.int32, device="cuda")
        ring = guard[16:24]
        ring.copy_(ints([3, 4, 5, 6, 50, -2, 0, 1]))
        t, n = table.clone(), ints(lens)
        offsets, positions, slots, taken = ops.fine_plan_packed(t, n, ints(new), ring, ints(span), 16, 40)
        assert (guard[:16] == 77).all() and (guard[24:] == 77).all()
        assert (slots >= -1).all() and (slots < 8 * 16).all() and (offsets.diff() >= 0).all() and (offsets <= 40).all() and ((n >= 0) & (n <= 64)).all()


def test_captured_plans(gpu):
    pool, new = Pool(6, 20, 90, 16, seed=3), ints([0] * 6)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.run(new, 400)
    torch.cuda.synchronize()
    pool.put()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = pool.run(new, 400)
    rng = random.Random(5)
    for _ in range(8):
        n = [rng.randrange(0, 60) for _ in range(6)]
        new.copy_(ints(n))
        graph.replay()
        torch.cuda.synchronize()
        want = pool.plan(n, 400)
        assert [g.tolist() for g in got] == list(want)
        pool.same()


# ---- filing --------------------------------------------------------------------------------------------------------------


def tables(n):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


@TYPES
@pytest.mark.parametrize("keep_keys", [True, False], ids=["kept", "filed"])
@pytest.mark.parametrize("case", [(32, 8, 16, 300), (8, 2, 48, 1), (0, 3, 32, 77), (5, 1, 128, 40), (64, 8, 16, 33)], ids=lambda c: "%d-%d-p%d-%d" % c)
def test_tokens_are_rotated_and_filed(gpu, case, keep_keys, dtype):
    n_q, Hkv, page, rows = case
    gen = torch.Generator().manual_seed(rows)
    n_pages, n_pos = rows // page + 4, 200
    cos, sin = tables(n_pos)
    big = torch.randn(rows, n_q + 2 * Hkv + 1, D, generator=gen).to(dtype).cuda()
    qkv = big[:, :n_q + 2 * Hkv]                      # (rows with something between them)
    kv = torch.full((n_pages, page, 2 * Hkv + 1, D), math.nan, dtype=dtype, device="cuda")[:, :, :2 * Hkv].transpose(1, 2)   # token-major
    slots = torch.randperm(n_pages * page, generator=gen)[:rows].to(torch.int32)
    positions = torch.randint(0, 300, (rows,), generator=gen).to(torch.int32)   # (some behind the table: its last row)
    if rows > 10:
        positions[[2, rows - 1]] = ints([-1, -40]).cpu()
        slots[[2, 5, 6, 7]] = ints([3, -1, n_pages * page, 2147483647]).cpu()
    weights, where = torch.full((n_pages, Hkv, page), 3.0, device="cuda"), torch.full((n_pages, Hkv, page), -7, dtype=torch.int32, device="cuda")
    before, x = big.clone(), qkv.double()
    want_kv, want_w, want_p = kv.clone(), weights.clone(), where.clone()
    ops.fine_rope_packed(qkv, kv, slots.cuda(), cos, sin, positions.cuda(), n_q, weights=weights, key_positions=where, keep_keys=keep_keys)
    at = positions.clamp(0, n_pos - 1).long().cuda()
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    lo, hi = x[..., :64], x[..., 64:]
    y = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
    size = torch.cat((lo.abs() * c.abs() + hi.abs() * s.abs(),) * 2, -1)
    token = (positions >= 0).cuda()
    turned = torch.zeros(n_q + 2 * Hkv, dtype=torch.bool, device="cuda")
    turned[:n_q + (Hkv if keep_keys else 0)] = True
    # three roundings in 32 bits, one to the element type (in fp16 below 2^-14 half of 2^-24)
    bound = HALF_STEP[dtype] * (y.abs() + 1e-6 * size) + 4 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == torch.float16 else 0)
    changed = token[:, None] & turned
    assert ((qkv.double() - y).abs() <= bound)[changed].all()
    assert torch.equal(qkv[~changed], before[:, :n_q + 2 * Hkv][~changed]) and torch.equal(big[:, -1], before[:, -1])
    for t in range(rows):
        slot = int(slots[t])
        if positions[t] < 0 or not 0 <= slot < n_pages * page:
            continue
        p, r = slot // page, slot % page
        assert ((kv[p, :Hkv, r].double() - y[t, n_q:n_q + Hkv]).abs() <= bound[t, n_q:n_q + Hkv]).all()
        assert torch.equal(kv[p, Hkv:, r], before[t, n_q + Hkv:n_q + 2 * Hkv])
        if keep_keys:
            assert torch.equal(kv[p, :Hkv, r], qkv[t, n_q:n_q + Hkv])
        want_kv[p, :, r], want_w[p, :, r], want_p[p, :, r] = kv[p, :, r], 0.0, int(positions[t])
    assert torch.equal(kv.nan_to_num(9.0), want_kv.nan_to_num(9.0)) and torch.equal(weights, want_w) and torch.equal(where, want_p)


def test_filing_without_an_account_is_that_of_a_padded_batch(gpu):
    """One sequence: the bits of fine_rope_paged."""
    gen = torch.Generator().manual_seed(1)
    qkv = torch.randn(50, 48, D, generator=gen).half().cuda()
    kv, kv2 = torch.zeros(6, 16, 16, D, dtype=torch.float16, device="cuda"), torch.zeros(6, 16, 16, D, dtype=torch.float16, device="cuda")
    table, (cos, sin) = ints([[4, 0, 3, 1]]), tables(100)
    positions = torch.arange(7, 57, dtype=torch.int32, device="cuda")
    other = qkv.clone()[None]
    ops.fine_rope_paged(other, kv2, table, ints([60]), cos, sin, positions, 32, keep_keys=True)
    key = torch.arange(10, 60, device="cuda")
    ops.fine_rope_packed(qkv, kv, (table[0][key // 16] * 16 + key % 16).int(), cos, sin, positions, 32)
    assert torch.equal(qkv, other[0]) and torch.equal(kv, kv2)
