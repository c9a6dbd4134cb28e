"""Drafts of different sizes, from the plan to the accepted path: sequences that draft fewer tokens than the call has rows, none, or find no pages."""
import math

import pytest
import torch

import fmha_unified
from reference64 import D, attention64, check
from test_packed_gpu import Pool, TYPES, ints, tables
from test_tree_gpu import a_tree, descent, mask

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu


@TYPES
@pytest.mark.parametrize("S", [5, 33])
def test_drafts_of_different_sizes(gpu, S, dtype):
    B, Hq, Hkv, page, columns, n_pages = 6, 8, 2, 16, 12, 30
    gen = torch.Generator().manual_seed(S)
    pool = Pool(B, columns, n_pages, page, seed=3)
    pool.texts = [0] * B
    pool.put()
    kv = torch.full((n_pages, 2 * Hkv, page, D), math.nan, dtype=dtype, device="cuda")
    cos, sin = tables(400)

    # prompts of five sequences, one slot is empty; they leave 30 - 22 pages, which do not suffice for the drafts of all
    prompts = [50, 0, 130, 17, 64, 63]
    offsets, positions, slots, taken = pool.step(prompts, sum(prompts))
    qkv = torch.randn(sum(prompts), Hq + 2 * Hkv, D, generator=gen).to(dtype).cuda()
    ops.fine_rope_packed(qkv, kv, slots, cos, sin, positions, Hq)
    at = offsets.tolist()
    texts = [list(qkv[at[b]:at[b + 1], Hq:]) for b in range(B)]

    for round_ in range(4):
        drafted = [S, 0, max(S - 2, 1), 1, S, (S * (round_ + 1)) // 2]
        trees = [a_tree("some", S, 10 * round_ + b) for b in range(B)]
        depths = torch.tensor([descent(t, S).sum(1).tolist() for t in trees], dtype=torch.int32, device="cuda") - 1
        seq_lens, next_positions = pool.d[0], pool.d[3].clone()
        before = list(pool.lens)
        drafted = [min(n, S) for n in drafted]
        pool.texts, texts_before = None, pool.texts          # (the plan of a draft leaves the positions alone)
        ring, span = pool.d[1], pool.d[2]
        got = ops.fine_plan_packed(pool.d_table, seq_lens, ints(drafted), ring, span, page, B * S)
        want = pool.plan(drafted, B * S)
        taken = got[3]
        assert taken.tolist() == want[3]
        pool.texts = texts_before
        pool.same()
        assert seq_lens.tolist() == [n + t for n, t in zip(before, want[3])]

        qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=gen).to(dtype).cuda()
        ops.fine_rope_paged(qkv, kv, pool.d_table, seq_lens, cos, sin, next_positions[:, None] + depths, Hq, new_lens=taken, keep_keys=True)
        o, lse = ops.fine_fmha_tree_with_lse(qkv[:, :, :Hq].transpose(1, 2), kv, pool.d_table, seq_lens, ints(trees), new_lens=taken)
        paths = []
        for b in range(B):
            n, new = before[b], want[3][b]
            drafts = list(qkv[b, :new, Hq:])
            keys = texts[b] + drafts
            if keys:
                x = torch.stack(keys)
                check(o[b], lse[b], attention64(qkv[b, :, :Hq].transpose(0, 1), x[:, :Hkv].transpose(0, 1).contiguous(), x[:, Hkv:].transpose(0, 1).contiguous(),
                                                mask(trees[b], S, new, n + new)))
            else:
                assert (o[b] == 0).all() and (lse[b] == -math.inf).all()
            path, i = [], new - 1
            while i >= 0:
                path.insert(0, i)
                i = trees[b][i]
            paths.append(path)
            texts[b] = texts[b] + [drafts[i] for i in path]
        kept = ops.fine_keep_path(kv, pool.d_table, seq_lens, taken, ints([p + [-1] * (S - len(p)) for p in paths]))
        assert kept.tolist() == [n + len(p) for n, p in zip(before, paths)]
        pool.d[3].copy_(next_positions + kept - (seq_lens - taken))
        seq_lens.copy_(kept)
        pool.lens, pool.texts = kept.tolist(), pool.d[3].tolist()
        assert pool.texts == pool.lens
        if S == 33 and round_ == 0:
            assert any(t < n for t, n in zip(want[3], drafted))   # one found no pages


def test_drafts_that_are_planned_and_filed_in_a_captured_step(gpu):
    """One graph for drafts of any sizes up to S."""
    B, S, Hq, Hkv, page, columns, n_pages = 3, 9, 8, 2, 16, 8, 24
    gen = torch.Generator().manual_seed(1)
    cos, sin = tables(200)
    trees = ints([a_tree("some", S, b) for b in range(B)])
    depths = torch.tensor([descent(t, S).sum(1).tolist() for t in trees.tolist()], dtype=torch.int32, device="cuda") - 1
    state = [torch.full((B, columns), -1, dtype=torch.int32, device="cuda"), ints([0] * B), torch.arange(n_pages, dtype=torch.int32, device="cuda"), ints([0, n_pages]), ints([0] * B)]
    drafted, qkv = ints([0] * B), torch.zeros(B, S, Hq + 2 * Hkv, D, dtype=torch.float16, device="cuda")
    kv = torch.zeros(n_pages, 2 * Hkv, page, D, dtype=torch.float16, device="cuda")
    path = ints([[0] + [-1] * (S - 1)] * B)

    def step(table, seq_lens, ring, span, positions, kv, qkv):
        taken = ops.fine_plan_packed(table, seq_lens, drafted, ring, span, page, B * S)[3]
        ops.fine_rope_paged(qkv, kv, table, seq_lens, cos, sin, positions[:, None] + depths, Hq, new_lens=taken)
        o = ops.fine_fmha_tree(qkv[:, :, :Hq].transpose(1, 2), kv, table, seq_lens, trees, new_lens=taken)
        kept = ops.fine_keep_path(kv, table, seq_lens, taken, path)
        positions += kept - (seq_lens - taken)
        seq_lens.copy_(kept)
        return o

    other, kv2 = [x.clone() for x in state], kv.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*[x.clone() for x in state], kv.clone(), qkv.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = step(*state, kv, qkv)
    for sizes in ([9, 3, 0], [1, 9, 9], [0, 0, 0], [9, 0, 1], [5, 9, 9]):
        x = torch.randn(qkv.shape, generator=gen).half().cuda()
        drafted.copy_(ints(sizes))
        qkv.copy_(x)
        graph.replay()
        want = step(*other, kv2, x)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(kv, kv2) and torch.equal(qkv, x)
        assert all(torch.equal(a, b) for a, b in zip(state, other))
        assert state[1].tolist() == state[4].tolist()
