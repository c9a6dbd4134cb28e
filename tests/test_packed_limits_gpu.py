"""Packed batches and drafts of as many sequences as a call takes, or of many more than have rows."""
import math
import random

import pytest
import torch

import fmha_unified
from test_packed_gpu import Pool, batch, check_packed, ints, offsets_of
from test_paged_gpu import Cache, queries
from test_tree_gpu import a_tree, check_tree

ops = fmha_unified.ops
pytestmark = pytest.mark.gpu


def test_a_plan_of_as_many_sequences_as_a_call_takes(gpu):
    pool = Pool(65535, 3, 100000, 16)
    rng = random.Random(0)
    for most in (40, 3, 9):
        new = [rng.randrange(most) for _ in range(65535)]
        pool.step(new, sum(new) - 1000 if most == 9 else sum(new) + 3)


def test_prompts_of_more_sequences_than_rows(gpu):
    rng = random.Random(1)
    lens = [0] * 100000
    for i in rng.sample(range(100000), 300):
        lens[i] = rng.randrange(1, 9)
    lens[77777] = 500
    q, k, v = batch(lens, 8, 2, torch.bfloat16, spare=11)
    o, lse = ops.fine_fmha_packed_with_lse(q, k, v, offsets_of_many(lens))
    check_packed(q, k, v, [n for n in lens if n], o, lse)


def offsets_of_many(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(lens).cumsum(0)]).int().cuda()


@pytest.mark.parametrize("S", [3, 20], ids=["few", "many"])
def test_trees_of_many_sequences(gpu, S):
    lens = [(37 * i) % 97 + S for i in range(600)]
    new = [(7 * i) % (S + 1) for i in range(600)]
    cache = Cache(lens, 2, 16, dtype=torch.float16)
    q = queries(cache, 8, S)
    trees = [a_tree("some", S, b) for b in range(600)]
    o, lse = ops.fine_fmha_tree_with_lse(q, *cache.args, ints(trees), new_lens=ints(new))
    check_tree(cache, q, trees, o, lse, new)
