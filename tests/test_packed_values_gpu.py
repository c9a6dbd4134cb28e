"""Infinities and NaN among the values of packed prompts: where they are and what they cost.

A row that does not see such a value has the output that it has with a zero in its place, bit by bit: the weight is zero either way. A row that sees some
has, in their columns, what the sum is with them: NaN where one is NaN or two are infinite with different signs, otherwise the infinity, since every weight is
positive. (A weight is no number, or zero, where its key is not finite: an infinity times that is NaN.)"""
import math

import pytest
import torch

import fmha_unified
from reference64 import D
from test_packed_gpu import TYPES, batch, offsets_of, pinned

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu


def seen_of(v, lens, causal, bad_keys=None):
    """For every row, kv head and column: whether a NaN, +infinity, -infinity is among the values that the row sees."""
    kinds = [v.isnan(), v == math.inf, v == -math.inf]
    if bad_keys is not None:   # [rows, Hkv]
        kinds = [kinds[0] | (v.isinf() & bad_keys[..., None]), kinds[1] & ~bad_keys[..., None], kinds[2] & ~bad_keys[..., None]]
    out, at = [torch.zeros_like(kinds[0]) for _ in kinds], 0
    for n in lens:
        rows = slice(at, at + n)
        for x, y in zip(out, kinds):
            if n:
                x[rows] = y[rows].cummax(0).values if causal else y[rows].any(0, keepdim=True)
        at += n
    return out


def check_values(q, k, v, lens, causal, call, bad_keys=None):
    clean = torch.where(v.isfinite(), v, torch.zeros_like(v))
    o, lse = call(q, k, v, causal)
    want, want_lse = call(q, k, clean, causal)
    assert want[: sum(lens)].isfinite().all()
    group = q.shape[1] // k.shape[1]
    nan, above, below = (x.repeat_interleave(group, 1) for x in seen_of(v, lens, causal, bad_keys))
    nan |= above & below
    want = torch.where(above, math.inf, want.float())
    want = torch.where(below, -math.inf, want)
    want = torch.where(nan, math.nan, want)
    rows = slice(0, sum(lens))
    assert torch.equal(lse[:, rows], want_lse[:, rows])
    assert torch.equal(o[rows].float().nan_to_num(nan=7e30, posinf=8e30, neginf=-8e30), want[rows].nan_to_num(nan=7e30, posinf=8e30, neginf=-8e30))
    assert (o[sum(lens):] == 0).all() and (lse[:, sum(lens):] == -math.inf).all()


def spoil(v, lens, how, seed=0):
    """Infinities and NaN in some of the values."""
    gen, at = torch.Generator().manual_seed(seed), 0
    r = lambda n: int(torch.randint(n, (1,), generator=gen))
    kinds = (math.nan, math.inf, -math.inf)
    v = v.clone()
    if how in ("few", "many"):
        x = torch.rand(v.shape, generator=gen)
        share = 3e-5 if how == "few" else 0.02
        for i, kind in enumerate(kinds):
            v[((x > i * share) & (x <= (i + 1) * share)).cuda()] = kind
        return v
    for i, n in enumerate(lens):
        if n:
            if how == "one":        # an element
                v[at + r(n), r(v.shape[1]), r(D)] = kinds[i % 3]
            elif how == "ends":     # the first and the last key of a sequence
                v[at + n - 1, :, r(D)] = kinds[i % 3]
                v[at, :, r(D)] = kinds[(i + 1) % 3]
            elif how == "tiles":    # around the borders of tiles
                for j in (63, 64, 65, 127, 128, 255, 256, 511, 512):
                    if j < n:
                        v[at + j, r(v.shape[1]), r(D)] = kinds[r(3)]
            elif how == "rows":     # whole rows
                v[at + r(n), r(v.shape[1])] = math.nan
                v[at + r(n), r(v.shape[1])] = math.inf
        at += n
    return v


CASES = [   # Hq, Hkv, lengths: items of every number of heads side by side, one and several a workgroup, found by the workgroup and in a list
    (8, 2, [70, 300, 513, 9]),
    (32, 8, [300 + (163 * i) % 701 for i in range(16)]),
    (12, 4, [(53 * i) % 150 for i in range(65)]),
    (64, 8, [200 + (97 * i) % 300 for i in range(70)]),
    (16, 16, [1000, 30, 700, 1, 64, 129]),
    (16, 8, [513, 129, 64, 33, 1100, 900, 1300]),
    (32, 8, [256] * 16),
    (1, 1, [2049]),
    (8, 8, [(7 * i) % 5 for i in range(5000)]),   # more items a workgroup than are worked out together
]


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("how", ["one", "ends", "tiles", "rows", "few", "many"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%d-%d-B%d-%d" % (c[0], c[1], len(c[2]), sum(c[2])))
def test_rows_have_what_they_see(gpu, case, how, causal, dtype):
    Hq, Hkv, lens = case
    q, k, v = batch(lens, Hq, Hkv, dtype, spare=3)
    v = spoil(v.contiguous(), lens, how)
    for variant in (1, 2):
        check_values(q, k, v, lens, causal, lambda q, k, v, causal: pinned(q, k, v, offsets_of(lens), causal, variant))


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_infinities_whose_weights_are_small(gpu, causal, dtype):
    """Weights down to about e^-60, which are zero in 16 bits."""
    lens = [700, 90]
    q, k, v = batch(lens, 16, 4, dtype, scale=1.0)
    q, k, v = (x.contiguous() for x in (q, k, v))
    q[:, :, 0], k[:, :, 0] = 26, 1
    for at in (0, 5, 64, 300, 699, 700, 789):
        k[at, :, 0] = -25
        v[at, at % 4, at % D] = math.inf if at % 2 else -math.inf
    for variant in (1, 2):
        check_values(q, k, v, lens, causal, lambda q, k, v, causal: pinned(q, k, v, offsets_of(lens), causal, variant))


@TYPES
def test_infinities_whose_keys_are_infinite(gpu, dtype):
    """A key whose scores are -infinity weighs nothing, and nothing times an infinity is NaN."""
    lens = [300, 700, 65]
    q, k, v = batch(lens, 16, 4, dtype, scale=0.5)
    q, k, v = (x.contiguous() for x in (q, k, v))
    q[:, :, 3] = q[:, :, 3].abs() + 0.25
    bad = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for at in (5, 100, 299, 300 + 70, 300 + 640, 1000 + 64):
        k[at, at % 4, 3] = -math.inf
        v[at, at % 4, at % D] = math.inf
        bad[at, at % 4] = True
    for variant in (1, 2):
        check_values(q, k, v, lens, True, lambda q, k, v, causal: pinned(q, k, v, offsets_of(lens), causal, variant), bad)


def test_captured_calls_see_the_values_of_each_replay(gpu):
    lens = [300 + (163 * i) % 701 for i in range(16)]
    q, k, v = batch(lens, 32, 8, torch.float16)
    q, k, v = (x.contiguous() for x in (q, k, v))
    clean, offsets, side = v.clone(), offsets_of(lens), torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.fine_fmha_packed_with_lse(q, k, v, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets)

    def replay(q, k, v_now, causal):
        v.copy_(v_now)
        graph.replay()
        return o.clone(), lse.clone()

    for i, how in enumerate(("one", "many", "ends", "few", "rows")):
        check_values(q, k, spoil(clean, lens, how, seed=i), lens, True, replay)


def test_two_streams_at_once(gpu):
    """Each with items that are worked out again."""
    lens = ([300 + (163 * i) % 701 for i in range(16)], [(53 * i) % 150 for i in range(65)])
    calls = []
    for seed, n in enumerate(lens):
        q, k, v = batch(n, 16, 4, torch.float16, seed=seed)
        calls.append((q, k, spoil(v.contiguous(), n, "few" if seed else "tiles", seed), offsets_of(n)))
    want = [ops.fine_fmha_packed_with_lse(*c) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((i, ops.fine_fmha_packed_with_lse(*calls[i])))
    torch.cuda.synchronize()
    for i, (o, lse) in got:
        assert torch.equal(o.nan_to_num(7.0), want[i][0].nan_to_num(7.0)) and torch.equal(o.isnan(), want[i][0].isnan()) and torch.equal(lse, want[i][1])


def times_of(*calls):
    """Of each the best of 15 runs of 5, in turn"""
    best = [math.inf] * len(calls)
    for _ in range(15):
        for i, call in enumerate(calls):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                call()
            b.record()
            torch.cuda.synchronize()
            best[i] = min(best[i], a.elapsed_time(b))
    return best


@pytest.mark.parametrize("where", [0, 500, 900])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_spoilt_value_costs_no_more_than_a_pass(gpu, value, where):
    """One element of prompts of 1000 tokens. All that it can ask for is one more pass over the values, without products, of the waves that see it."""
    lens = [1000] * 16
    q, k, v = batch(lens, 32, 8, torch.float16)
    q, k, v = (x.contiguous() for x in (q, k, v))
    clean, offsets = v.clone(), offsets_of(lens)
    for b in range(16):
        v[1000 * b + where, :, 5] = value
    call = lambda v: ops.fine_fmha_packed(q, k, v, offsets)
    call(clean), call(v)
    plain, spoilt = times_of(lambda: call(clean), lambda: call(v))
    print("%.3f" % (spoilt / plain))
    assert spoilt < 2 * plain
