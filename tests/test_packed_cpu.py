"""CPU-only checks of packed batches, drafted trees and accepted paths: what their entry points refuse, before anything is launched."""
import ctypes

import pytest
import torch

import fmha_unified
from test_paged_cpu import BAD_CACHES, P, Seen, cache, tensors

ops = fmha_unified.ops
BIG = 1 << 60   # a workspace that is large enough whatever it is asked to be


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join("%s=%s" % x for x in d.items()))
def test_tree_and_path_refuse_a_bad_cache(lib, bad):
    cdll, c = lib.load(), cache(lib, **dict(dict(new_lens=P), **bad))
    refused = (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED)
    assert cdll.mi355_cache_keep_path(c, P, 4, 4, P * 16, None) in refused and cdll.mi355_last_error()
    if set(bad) <= {"weights"}:
        return   # (a tree's call does not look at the account)
    assert cdll.mi355_fmha_paged_tree(c, P, P, P, 32, 4, None, P, 4, 0.1, P, BIG, None) in refused and cdll.mi355_last_error()


def test_tree_refuses_bad_arguments(lib):
    cdll, c = lib.load(), cache(lib)
    need = cdll.mi355_fmha_paged_tree_workspace_bytes(c, 32, 8)

    def call(Q=P, O=P, Hq=32, S=8, strides=None, parents=P, batch=8, scale=0.1, ws=P, size=BIG):
        st = None if strides is None else (ctypes.c_int64 * 6)(*strides)
        return cdll.mi355_fmha_paged_tree(c, Q, O, None, Hq, S, st, parents, batch, scale, ws, size, None)

    bad = [dict(Q=None), dict(O=None), dict(parents=None), dict(Q=P + 2), dict(O=P + 8), dict(Hq=31), dict(Hq=0), dict(S=0), dict(S=257, batch=257), dict(batch=7), dict(batch=-8),
           dict(scale=0.0), dict(scale=float("inf")), dict(strides=[8, 8, 4, 8, 8, 8]), dict(strides=[8, 8, 8, 8, 8, 8])]
    if need > 0:
        bad += [dict(ws=None), dict(size=need - 1), dict(ws=P + 8)]
    for kw in bad:
        assert call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw
    assert cdll.mi355_fmha_paged_tree(None, P, P, None, 32, 8, None, P, 8, 0.1, P, BIG, None) == lib.ERR_BAD_ARGUMENT
    assert cdll.mi355_fmha_paged_tree_workspace_bytes(cache(lib, page_size=0), 32, 8) == 0


def test_a_path_refuses_bad_arguments(lib):
    cdll, c = lib.load(), cache(lib, new_lens=P)

    def call(path=P, length=4, batch=4, out=P * 16, cc=c):
        return cdll.mi355_cache_keep_path(cc, path, length, batch, out, None)

    for kw in (dict(path=None), dict(out=None), dict(length=0), dict(length=(1 << 28) + 1), dict(batch=3), dict(batch=-4), dict(out=P), dict(out=P + 12),
               dict(cc=cache(lib, new_lens=None)), dict(cc=cache(lib, new_lens=P * 16 + 8))):
        assert call(**kw) == lib.ERR_BAD_ARGUMENT, kw


def test_a_plan_refuses_bad_arguments(lib):
    cdll = lib.load()
    names = ("table", "stride", "lens", "new", "next", "ring", "span", "B", "columns", "n_pages", "page", "rows", "offsets", "positions", "slots", "taken", "ws", "size")
    good = dict(zip(names, (P, 8, P, P, 2 * P, P, P, 4, 8, 32, 16, 100, P, P, P, P, P, BIG)))

    def call(**kw):
        return cdll.mi355_packed_plan(*dict(good, **kw).values(), None)

    need = cdll.mi355_packed_plan_workspace_bytes(4)
    assert need > 0 and cdll.mi355_packed_plan_workspace_bytes(0) == 0 and cdll.mi355_packed_plan_workspace_bytes(65536) == 0
    for kw in ([{n: None} for n in ("table", "lens", "new", "ring", "span", "offsets", "positions", "slots", "taken", "ws")] +
               [dict(B=0), dict(columns=0), dict(n_pages=0), dict(rows=-1), dict(page=0), dict(page=24), dict(stride=7), dict(size=need - 1), dict(ws=P + 8), dict(B=65536),
                dict(rows=(1 << 28) + 1), dict(next=P + 12, lens=P), dict(columns=(1 << 24) + 1, stride=1 << 25), dict(n_pages=1 << 27, page=16), dict(B=60000, columns=1 << 16, stride=1 << 16)]):
        assert call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw


def test_filing_a_packed_batch_refuses_bad_arguments(lib):
    cdll, row = lib.load(), 48 * 128

    def call(qkv=P, rows=4, q_heads=32, x_row=row, cos=P, sin=P, pos=P, slots=P, n=100, **pool):
        return cdll.mi355_rope_packed(cache(lib, **dict(dict(block_table=None, seq_lens=None, B=0, max_pages=0), **pool)), qkv, rows, q_heads, 1, x_row, cos, sin, pos, slots, n, None)

    for kw in (dict(qkv=None), dict(cos=None), dict(sin=None), dict(pos=None), dict(slots=None), dict(pages=None), dict(qkv=P + 2), dict(cos=P + 4), dict(rows=0), dict(rows=1 << 24),
               dict(q_heads=-1), dict(n=0), dict(x_row=row - 8), dict(x_row=row + 4), dict(dtype=2), dict(Hkv=0), dict(n_pages=0), dict(page_size=24), dict(n_pages=1 << 27),
               dict(page_stride=0), dict(row_stride=129), dict(row_stride=1 << 24), dict(weights=P + 4), dict(key_positions=P + 8), dict(pages=P + 8)):
        assert call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw


def test_packed_attention_refuses_bad_arguments(lib):
    cdll = lib.load()
    need = cdll.mi355_fmha_packed_workspace_bytes(100, 3, 32, 8)
    assert need > 0

    def call(Q=P, K=P, V=P, O=P, offsets=P, rows=100, B=3, Hq=32, Hkv=8, strides=None, scale=0.1, dtype=0, ws=P, size=BIG):
        st = None if strides is None else (ctypes.c_int64 * 8)(*strides)
        return cdll.mi355_fmha_packed(Q, K, V, O, None, offsets, rows, B, Hq, Hkv, st, scale, 1, dtype, ws, size, None)

    dense = [4096, 128, 1024, 128, 1024, 128, 4096, 128]
    for kw in ([{n: None} for n in ("Q", "K", "V", "O", "offsets", "ws")] + [{n: P + 8} for n in ("Q", "K", "V", "O", "ws")] +
               [dict(rows=0), dict(B=0), dict(Hq=0), dict(Hkv=0), dict(Hq=31), dict(scale=0.0), dict(scale=3e38), dict(dtype=2), dict(size=need - 1),
                dict(rows=(1 << 28) + 1), dict(rows=1 << 28, Hq=4096), dict(B=1 << 27, rows=1 << 27)] +
               [dict(strides=dense[:i] + [x] + dense[i + 1:]) for i in range(8) for x in (-8, 4)] + [dict(strides=dense[:i] + [1 << 24] + dense[i + 1:]) for i in (0, 2, 4, 6)] +
               [dict(strides=dense[:6] + [64, 128]), dict(strides=dense[:6] + [4096, 0])]):
        assert call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw
    for sizes in ((0, 3, 32, 8), (100, 0, 32, 8), (100, 3, 4, 8), (1 << 28, 3, 4096, 8), (100, 3, 32, 0)):
        assert cdll.mi355_fmha_packed_workspace_bytes(*sizes) == 0
    assert cdll.mi355_internal_fmha_packed_variant(P, P, P, P, None, P, 100, 3, 32, 8, None, 0.1, 1, 0, P, BIG, 3, None) == lib.ERR_BAD_ARGUMENT


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_operators_refuse_what_is_not_on_the_gpu_and_wrong_shapes():
    t, h = tensors(S=4), torch.float16
    pool = (t["kv_pages"], t["block_table"], t["seq_lens"])
    qkv, table = torch.zeros(6, 12, 128, dtype=h), torch.ones(50, 64)
    for call in (lambda: ops.fine_fmha_tree(t["q"], *pool, ints(2, 4)), lambda: ops.fine_keep_path(*pool, ints(2), ints(2, 3)),
                 lambda: ops.fine_plan_packed(t["block_table"], ints(2), ints(2), ints(5), ints(2), 16, 10),
                 lambda: ops.fine_rope_packed(qkv, t["kv_pages"], ints(6), table, table, ints(6), 8),
                 lambda: ops.fine_fmha_packed(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], ints(3))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    q, k = qkv[:, :8], qkv[:, 8:10]
    for match, args in (("dtype|float16", (q.float(), k.float(), k.float())), ("128", (q[..., :64], k, k)), ("q's rows", (q, k[:5], k[:5])), ("one shape", (q, k, k[:, :1])),
                        ("multiple of kv heads", (q[:, :7], k, k)), ("empty", (q[:0], k[:0], k[:0])), ("q's dtype", (q, k.bfloat16(), k)), ("heads, 128", (q[0], k[0], k[0]))):
        with pytest.raises(RuntimeError, match=match):
            ops.fine_fmha_packed(*args, ints(3))


def test_operators_name_what_they_write():
    for name, written in (("fmha_tree", []), ("fmha_tree_lse", []), ("keep_path", ["kv_pages", "weights", "key_positions"]), ("fmha_packed", []), ("fmha_packed_lse", []),
                          ("plan_packed", ["block_table", "seq_lens", "free_pages", "free_span", "next_positions"]),
                          ("rope_packed", ["qkv", "kv_pages", "weights", "key_positions"])):
        schema = getattr(torch.ops.fmha_unified, name).default._schema
        assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == written


def test_what_watches_the_dispatcher_sees_the_functions():
    t, one = tensors(S=4), torch.ones(50, 64)
    pool = (t["kv_pages"], t["block_table"], t["seq_lens"])
    qkv = torch.zeros(6, 12, 128, dtype=torch.float16)
    with Seen() as seen:
        ops.fine_fmha_tree(t["q"], *pool, ints(4))
        ops.fine_fmha_tree_with_lse(t["q"], *pool, ints(2, 4), new_lens=ints(2))
        ops.fine_keep_path(*pool, ints(2), ints(2, 3))
        try:
            ops.fine_plan_packed(t["block_table"], ints(2), ints(2), ints(5), ints(2), 16, 10)
        except TypeError:
            pass   # (the mode's answer is no tuple of four)
        ops.fine_rope_packed(qkv, t["kv_pages"], ints(6), one, one, ints(6), 8)
        ops.fine_fmha_packed(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], ints(3))
        ops.fine_fmha_packed_with_lse(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], ints(3), causal=False)
    wanted = ["fmha_tree", "fmha_tree_lse", "keep_path", "plan_packed", "rope_packed", "fmha_packed", "fmha_packed_lse"]
    assert [n for n in seen.names if n.startswith("fmha_unified")] == ["fmha_unified::" + n for n in wanted]
