"""Trees of drafted tokens over a cache in pages, and their accepted paths, against plain loops in 64 bits; and a run of packed prompts, drafts and steps."""
import math

import pytest
import torch

import fmha_unified
from reference64 import D, attention64, check
from test_packed_gpu import Pool, TYPES, ints, tables
from test_paged_gpu import Cache, queries

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu


def a_tree(kind, S, seed):
    gen = torch.Generator().manual_seed(seed)
    if kind == "chain":
        return [i - 1 for i in range(S)]
    if kind == "roots":
        return [-1] * S
    if kind == "pairs":
        return [(i - 1) // 2 for i in range(S)]
    if kind == "wild":      # numbers that make roots among those that do not
        return [int(x) for x in torch.randint(-3, S + 5, (S,), generator=gen)]
    back = torch.randint(1, 9, (S,), generator=gen).tolist()
    return [max(-1, i - x) for i, x in enumerate(back)]


def descent(parents, S):
    """[S, S]: whether token j is token i or on its path to a root."""
    seen = torch.zeros(S, S, dtype=torch.bool)
    for i in range(S):
        j = i
        while True:
            seen[i, j] = True
            if not 0 <= parents[j] < j:
                break
            j = parents[j]
    return seen


def mask(parents, S, new, n):
    """[S, n]: what the rows see of the sequence's n keys."""
    seen = torch.zeros(S, n, dtype=torch.bool)
    base, down = n - new, descent(parents, S)
    for i in range(min(new, S)):
        seen[i, :max(base, 0)] = True
        for j in range(new):
            if base + j >= 0 and down[i, j]:
                seen[i, base + j] = True
    return seen.cuda()


def check_tree(cache, q, trees, o, lse, new=None, hidden=lambda b: None):
    S = q.shape[2]
    for b, n in enumerate(cache.seq_lens):
        k, v = (x.transpose(0, 1) for x in cache_keys(cache, b))
        seen = mask(trees[b], S, S if new is None else new[b], n)
        none = hidden(b)
        if none is not None:
            seen &= ~none
        check(o[b], lse[b], attention64(q[b], k, v, seen))


def cache_keys(cache, b):
    pg, sl = cache.at(b)
    x = cache.kv[pg, :, sl]
    return x[:, :cache.Hkv], x[:, cache.Hkv:]


TREES = [   # Hq, Hkv, S, page, lengths, new_lens, options
    (8, 2, 1, 16, [300], None, {}),
    (8, 2, 26, 16, [300], None, {}),
    (8, 2, 7, 16, [7, 8, 300, 39], None, {}),                      # 28 columns; nothing in front of the draft
    (4, 4, 4, 16, [513, 4, 60, 1000], [4, 1, 0, 3], {}),           # few columns, a padded batch
    (4, 4, 16, 16, [16, 700, 31, 32, 33, 47, 48, 49], None, {}),
    (6, 3, 5, 48, [5, 700, 3, 0, 60], None, {}),                   # sequences shorter than their drafts
    (32, 8, 8, 32, [8191], None, {}),                              # 32 columns, cut
    (32, 8, 13, 32, [900, 77, 2049], [13, 5, 9], {}),              # 52 columns: two blocks
    (1, 1, 100, 16, [400, 131], None, {}),                         # one head, four blocks, a workgroup a pair
    (2, 2, 256, 16, [300, 256], None, dict(max_pages=20)),
    (32, 8, 64, 64, [4000], None, {}),                             # 256 columns
    (32, 8, 32, 32, [2000, 60, 333, 32], [32, 7, 1, 32], {}),
    (32, 8, 32, 16, [(537 * i) % 900 + 32 for i in range(20)], None, {}),
    (16, 2, 100, 16, [1500, 100, 731], [100, 3, 66], {}),
    (40, 8, 60, 128, [700, 90], None, dict(token_major=True)),
    (8, 1, 256, 32, [3000, 257, 200], None, {}),                   # 2048 columns
    (64, 8, 255, 32, [2500] * 9, None, {}),
    (32, 8, 8, 16, [300, 20], None, dict(max_pages=900)),
    (8, 4, 3, 16, [(37 * i) % 97 + 3 for i in range(70)], None, {}),
    (8, 2, 20, 16, [(37 * i) % 600 + 20 for i in range(70)], None, {}),     # more sequences than are ordered: a workgroup a triple
    (8, 1, 24, 16, [(191 * i) % 1500 for i in range(40)], [(7 * i) % 25 for i in range(40)], {}),   # some without keys, some without tokens
    (16, 2, 32, 32, [3000] + [40] * 20, None, {}),                         # one that is cut, and others
]


@TYPES
@pytest.mark.parametrize("kind, case", [(kind, case) for case in TREES for kind in ("some", "chain", "roots", "wild")[:2 if max(case[4]) > 1000 else 4]],
                         ids=lambda c: c if isinstance(c, str) else "%d-%d-S%d-p%d-B%d-%s" % (c[0], c[1], c[2], c[3], len(c[4]), max(c[4])))
def test_attention_of_a_tree(gpu, kind, case, dtype):
    Hq, Hkv, S, page, lens, new, options = case
    cache = Cache(lens, Hkv, page, dtype, **options)
    q = queries(cache, Hq, S)
    if new is not None:
        for b, n in enumerate(new):
            q[b, :, n:] = math.nan     # rows that are no tokens
    trees = [a_tree(kind, S, b) for b in range(len(lens))]
    lens_arg = None if new is None else ints(new)
    o, lse = ops.fine_fmha_tree_with_lse(q, *cache.args, ints(trees), new_lens=lens_arg)
    assert o.shape == q.shape and o.is_contiguous() and lse.shape == q.shape[:3]
    check_tree(cache, q, trees, o, lse, new)
    again = ops.fine_fmha_tree(q, *cache.args, ints(trees), new_lens=lens_arg)
    assert torch.equal(o, again)
    if kind == "chain":   # what fine_fmha_paged's rows see
        check_tree(cache, q, trees, *ops.fine_fmha_paged_with_lse(q, *cache.args, new_lens=lens_arg), new)


@TYPES
def test_one_tree_for_all_sequences(gpu, dtype):
    cache = Cache([700, 40, 90], 8, 32, dtype)
    q, tree = queries(cache, 32, 20), a_tree("pairs", 20, 0)
    o, lse = ops.fine_fmha_tree_with_lse(q, *cache.args, ints(tree))
    check_tree(cache, q, [tree] * 3, o, lse)
    assert torch.equal(o, ops.fine_fmha_tree(q, *cache.args, ints([tree] * 3)))


@TYPES
@pytest.mark.parametrize("case", [(8, 2, 4), (8, 2, 7), (32, 8, 8), (8, 2, 40), (32, 8, 64), (8, 1, 200)], ids=lambda c: "%d-%d-S%d" % c)
def test_what_a_drafted_token_does_not_see_has_no_influence(gpu, case, dtype):
    """Infinities and NaN in the values and keys of drafted tokens: only those that descend from them know."""
    Hq, Hkv, S = case
    lens = [600, S + 3]
    cache = Cache(lens, Hkv, 16, dtype)
    q, trees = queries(cache, Hq, S, scale=0.2), [a_tree("some", S, 3), a_tree("pairs", S, 0)]
    for b, n in enumerate(lens):
        pg, sl = cache.at(b)
        last, mid = n - 1, n - 1 - S // 3
        cache.kv[pg[mid], Hkv, sl[mid], 3] = math.inf
        cache.kv[pg[last], :, sl[last]] = math.nan
    o, lse = ops.fine_fmha_tree_with_lse(q, *cache.args, ints(trees))
    # (the last token itself is NaN throughout)
    assert o[:, :, -1].isnan().all() and lse[:, :, -1].isnan().all()
    seen_rows = slice(0, S - 1)
    for b, n in enumerate(lens):
        k, v = (x.transpose(0, 1)[:, :-1] for x in cache_keys(cache, b))
        seen = mask(trees[b], S, S, n)[seen_rows, :-1]
        check(o[b][:, seen_rows], lse[b][:, seen_rows], attention64(q[b][:, seen_rows], k, v, seen))


@TYPES
@pytest.mark.parametrize("S", [4, 40], ids=["few", "many"])
def test_pages_outside_the_pool_hold_no_keys(gpu, S, dtype):
    cache = Cache([500, 100], 2, 16, dtype)
    q, trees = queries(cache, 8, S), [a_tree("some", S, b) for b in range(2)]
    holes = {0: [3, 30], 1: [0, 5]}
    table = cache.table.clone()
    for b, columns in holes.items():
        table[b, columns] = ints([-1, 1 << 30])
    o, lse = ops.fine_fmha_tree_with_lse(q, cache.kv, table, cache.lens, ints(trees))

    def hidden(b):
        none = torch.zeros(cache.seq_lens[b], dtype=torch.bool, device="cuda")
        for c in holes[b]:
            none[16 * c:16 * c + 16] = True
        return none

    check_tree(cache, q, trees, o, lse, hidden=hidden)


@pytest.mark.parametrize("Hq", [2, 8, 32], ids=["12-columns", "48-columns", "192-columns"])
def test_captured_trees(gpu, Hq):
    cache = Cache([900, 300], 2, 16)
    q, parents, new = queries(cache, Hq, 12), ints([a_tree("some", 12, b) for b in range(2)]), ints([12, 12])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.fine_fmha_tree_with_lse(q, *cache.args, parents, new_lens=new)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o, lse = ops.fine_fmha_tree_with_lse(q, *cache.args, parents, new_lens=new)
    for step, (lens, n) in enumerate((([900, 300], [12, 12]), ([100, 0], [3, 0]), ([12, 299], [12, 1]), ([899, 17], [5, 12]))):
        cache.lens.copy_(ints(lens))
        cache.seq_lens = list(lens)
        new.copy_(ints(n))
        trees = [a_tree("wild" if step % 2 else "some", 12, 10 * step + b) for b in range(2)]
        parents.copy_(ints(trees))
        graph.replay()
        want = ops.fine_fmha_tree_with_lse(q, *cache.args, parents, new_lens=new)
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        check_tree(cache, q, trees, o, lse, n)


def test_trees_on_two_streams_at_once(gpu):
    """Each with parts of its own on their way through a workspace of its own."""
    calls = []
    for lens, S in (([900, 300], 12), ([2000, 5, 700], 40)):
        cache = Cache(lens, 2, 16)
        q, trees = queries(cache, 16, S), ints([a_tree("some", S, b) for b in range(len(lens))])
        calls.append((lambda c=cache, q=q, t=trees: ops.fine_fmha_tree_with_lse(q, *c.args, t), torch.cuda.Stream()))
    want = [call() for call, _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (call, stream) in enumerate(calls):
            with torch.cuda.stream(stream):
                got[i].append(call())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1]) for o, lse in got[i])


def test_pages_that_lie_beyond_32_bits(gpu):
    """Pages 2^23 elements apart, 5 GB from first to last."""
    small = Cache([700, 90], 2, 16)
    n_pages = 320
    whole = torch.empty(n_pages << 23, dtype=torch.float16, device="cuda")
    far = torch.as_strided(whole, (n_pages, 4, 16, D), (1 << 23, 16 * D, D, 1))
    far[-small.kv.shape[0]:].copy_(small.kv)
    table = small.table + (n_pages - small.kv.shape[0]) * (small.table >= 0)
    for S in (6, 60):
        q, trees = queries(small, 8, S), ints([a_tree("some", S, b) for b in range(2)])
        a, b = ops.fine_fmha_tree_with_lse(q, *small.args, trees), ops.fine_fmha_tree_with_lse(q, far, table.int(), small.lens, trees)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    path = ints([[0, 5, 6, 50], [1, 3, -1, -1]])
    ops.fine_keep_path(*small.args, ints([60, 60]), path)
    ops.fine_keep_path(far, table.int(), small.lens, ints([60, 60]), path)
    assert torch.equal(far[-small.kv.shape[0]:].nan_to_num(9.0), small.kv.nan_to_num(9.0))


# ---- accepted paths ----------------------------------------------------------------------------------------------------


def kept(path, n, length):
    """Places of the accepted tokens: `path` as far as it ascends and names drafted tokens that are keys."""
    got, missing = [], max(n - length, 0)
    for i in path:
        if not (got[-1] if got else missing - 1) < i < n:
            break
        got.append(i)
    return got


PATHS = [   # Hkv, page, lengths, new_lens, paths
    (2, 16, [300], [26], [[0, 2, 3, 9, 20]]),
    (8, 32, [700, 64, 65, 40, 64], [64, 64, 64, 40, 1], [[1, 2, 3, 63], [0, 1, 2, 3], [63], [-1, 5], [0]]),
    (1, 48, [100, 100, 100, 5, 0], [10, 10, 0, 9, 4], [[9], [3, 3, 4], [0, 1], [2, 3, 4, 6, 8], [0, 1]]),   # no path, a path that stops, drafts longer than their sequences
    (20, 16, [900] * 3, [200] * 3, [list(range(1, 200)), list(range(0, 200, 3)), list(range(100, 200))]),
    (3, 128, [513], [130], [[0, 5, 4, 7]]),
]


@TYPES
@pytest.mark.parametrize("account", [False, True], ids=["plain", "account"])
@pytest.mark.parametrize("case", PATHS, ids=lambda c: "%d-p%d-B%d-%d" % (c[0], c[1], len(c[2]), max(c[3])))
def test_accepted_paths_close_ranks(gpu, case, account, dtype):
    Hkv, page, lens, new, paths = case
    cache = Cache(lens, Hkv, page, dtype, token_major=Hkv == 3)
    cache.positions = torch.randint(0, 1000, cache.positions.shape, device="cuda", dtype=torch.int32)
    width = max(len(p) for p in paths) + 1
    given = ints([p + [-1] * (width - len(p)) for p in paths])
    want_kv, want_w, want_p = cache.kv.clone(), cache.weights.clone(), cache.positions.clone()
    left = []
    for b, path in enumerate(paths):
        base, accepted = lens[b] - new[b], kept(path, new[b], lens[b])
        pg, sl = cache.at(b)
        for j, i in enumerate(accepted):
            to, at = max(base, 0) + j, base + i
            for want, have in ((want_kv, cache.kv), (want_w, cache.weights), (want_p, cache.positions)):
                want[pg[to], :, sl[to]] = have[pg[at], :, sl[at]]
        left.append(max(base, 0) + len(accepted))
    more = dict(weights=cache.weights, key_positions=cache.positions) if account else {}
    before = cache.lens.clone()
    got = ops.fine_keep_path(*cache.args, ints(new), given, **more)
    assert got.tolist() == left and torch.equal(cache.lens, before)
    assert torch.equal(cache.kv.nan_to_num(9.0), want_kv.nan_to_num(9.0))
    if account:
        assert torch.equal(cache.weights.nan_to_num(9.0), want_w.nan_to_num(9.0)) and torch.equal(cache.positions, want_p)


def test_paths_leave_pages_outside_the_pool_alone(gpu):
    cache = Cache([64], 2, 16)
    table, before = cache.table.clone(), cache.kv.clone()
    table[0, 3] = -1                      # keys 48 .. 63: nothing comes from there
    got = ops.fine_keep_path(cache.kv, table, cache.lens, ints([40]), ints([[3, 30, 39]]))
    assert got.tolist() == [27]
    pg, sl = cache.at(0)
    before[pg[24], :, sl[24]] = before[pg[27], :, sl[27]]
    assert torch.equal(cache.kv.nan_to_num(9.0), before.nan_to_num(9.0))


def test_captured_paths(gpu):
    cache, lens = Cache([200, 90], 4, 16), [200, 90]
    start, path, new = cache.kv.clone(), ints([[-1] * 6] * 2), ints([0, 0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.fine_keep_path(*cache.args, new, path)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.fine_keep_path(*cache.args, new, path)
    for n, p in (([30, 20], [[0, 1, 9, 29, -1, -1], [5, 6, -1, -1, -1, -1]]), ([1, 64], [[0, -1, 2, 2, 2, 2], [3, 9, 20, 40, 50, 63]])):
        new.copy_(ints(n))
        path.copy_(ints(p))
        cache.kv.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        have = cache.kv.clone()
        cache.kv.copy_(start)
        want = ops.fine_keep_path(*cache.args, new, path)
        assert torch.equal(got, want) and torch.equal(have.nan_to_num(9.0), cache.kv.nan_to_num(9.0))
        assert got.tolist() == [lens[b] - n[b] + len(kept(p[b], n[b], lens[b])) for b in range(2)]


# ---- a run of them -------------------------------------------------------------------------------------------------------


@TYPES
def test_prompts_drafts_and_steps(gpu, dtype):
    """Prompts come packed; then rounds of a drafted tree, its accepted path and a step; one sequence ends and another takes its place. What each call attends to is
    checked against the texts kept on the side."""
    B, Hq, Hkv, page, columns = 4, 8, 2, 16, 16
    gen = torch.Generator().manual_seed(7)
    pool = Pool(B, columns, 50, page, seed=2)
    pool.texts = [0] * B
    pool.put()
    kv = torch.full((50, 2 * Hkv, page, D), math.nan, dtype=dtype, device="cuda")
    cos, sin = tables(400)
    texts = [[] for _ in range(B)]      # of each sequence: its keys and values, [2 Hkv, 128] each

    def project(rows):
        return torch.randn(rows, Hq + 2 * Hkv, D, generator=gen).to(dtype).cuda()

    def attended(b, q, seen):
        x = torch.stack(texts[b])
        return attention64(q, x[:, :Hkv].transpose(0, 1).contiguous(), x[:, Hkv:].transpose(0, 1).contiguous(), seen)

    def prompts(new, spare):
        rows = sum(new) + spare
        offsets, positions, slots, taken = pool.step(new, rows)
        assert taken.tolist() == new
        qkv = project(rows)
        ops.fine_rope_packed(qkv, kv, slots, cos, sin, positions, Hq)
        q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
        o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets)
        at = 0
        for b, n in enumerate(new):
            if n:
                texts[b] = list(qkv[at:at + n, Hq:])
                seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
                check(o[at:at + n].transpose(0, 1), lse[:, at:at + n], attended(b, q[at:at + n].transpose(0, 1), seen))
            at += n
        assert (o[at:] == 0).all()

    def draft(S, seed):
        trees = [a_tree("some", S, seed + b) for b in range(B)]
        depth = torch.tensor([descent(t, S).sum(1).tolist() for t in trees], dtype=torch.int32, device="cuda") - 1
        next_position = pool.d[3].clone()
        before = list(pool.lens)
        offsets, positions, slots, taken = pool.step([S] * B, B * S)
        positions = (next_position[:, None] + depth).reshape(-1)
        qkv = project(B * S)
        ops.fine_rope_packed(qkv, kv, slots, cos, sin, positions, Hq)
        q = qkv[:, :Hq].reshape(B, S, Hq, D).transpose(1, 2)
        o, lse = ops.fine_fmha_tree_with_lse(q, kv, pool.d_table, pool.d[0], ints(trees))
        paths = []
        for b in range(B):
            drafted = list(qkv[b * S:(b + 1) * S, Hq:])
            n = before[b]
            texts[b] += drafted
            check(o[b], lse[b], attended(b, q[b], mask(trees[b], S, S, n + S)))
            path, i = [], S - 1 - b
            while i >= 0:                                    # from some token to its root
                path.insert(0, i)
                i = trees[b][i]
            paths.append(path)
            texts[b] = texts[b][:n] + [drafted[i] for i in path]
        given = ints([p + [-1] * (S - len(p)) for p in paths])
        lens = ops.fine_keep_path(kv, pool.d_table, pool.d[0], ints([S] * B), given)
        assert lens.tolist() == [n + len(p) for n, p in zip(before, paths)]
        pool.d[0].copy_(lens)
        pool.d[3].copy_(next_position + lens - ints(before))
        pool.lens, pool.texts = lens.tolist(), pool.d[3].tolist()

    def step():
        offsets, positions, slots, taken = pool.step([1] * B, B)
        qkv = project(B)
        ops.fine_rope_packed(qkv, kv, slots, cos, sin, positions, Hq)
        q = qkv[:, :Hq].reshape(B, 1, Hq, D).transpose(1, 2)
        o, lse = ops.fine_fmha_paged_with_lse(q, kv, pool.d_table, pool.d[0])
        for b in range(B):
            texts[b].append(qkv[b, Hq:])
            check(o[b], lse[b], attended(b, q[b], torch.ones(1, len(texts[b]), dtype=torch.bool, device="cuda")))

    prompts([50, 1, 130, 17], 9)
    for i in range(4):
        draft((5, 12, 33, 1)[i], 10 * i)
        step()
    pool.lens[2] = 0                                         # this one is done
    pool.texts[2] = 0
    pool.put()
    texts[2] = []
    prompts([0, 0, 70, 0], 0)
    draft(9, 99)
    step()
