"""CPU-only checks of the paged key-value cache's entry points: what they refuse, before anything is launched."""
import ctypes

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import fmha_unified

ops = fmha_unified.ops
P = 0x10000   # an address that nothing reads


def cache(lib, **other):
    c = dict(pages=P, block_table=P, seq_lens=P, new_lens=None, weights=P, key_positions=P, page_stride=16 * 16 * 128, head_stride=16 * 128, row_stride=128,
             table_stride=8, n_pages=32, page_size=16, max_pages=8, B=4, Hkv=8, dtype=0)
    c.update(other)
    return lib.PagedKV(**c)


BAD_CACHES = [dict(pages=None), dict(block_table=None), dict(seq_lens=None), dict(pages=P + 8), dict(weights=P + 4), dict(key_positions=P + 8), dict(B=0), dict(Hkv=0), dict(n_pages=0), dict(max_pages=0),
              dict(page_size=0), dict(page_size=8), dict(page_size=24), dict(dtype=2), dict(table_stride=7), dict(page_stride=0), dict(head_stride=64),
              dict(row_stride=129), dict(row_stride=-128), dict(row_stride=1 << 24), dict(page_size=1 << 20, row_stride=1 << 20), dict(B=9000),
              dict(max_pages=(1 << 24) + 1, table_stride=1 << 25), dict(max_pages=1 << 22, table_stride=1 << 22, B=1000, Hkv=10)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "-".join("%s=%s" % x for x in d.items()))
def test_every_entry_point_refuses_a_bad_cache(lib, bad):
    cdll, c = lib.load(), cache(lib, **bad)
    big = 1 << 60   # a workspace that is large enough whatever it is asked to be
    for rc in (cdll.mi355_fmha_paged(c, P, P, P, 32, 1, None, 0.1, P, big, None),
               cdll.mi355_rope_paged(c, P, 1, 32, 0, 48 * 128, 48 * 128, P, P, P, 0, 100, None),
               cdll.mi355_fmha_key_weights(c, P, P, 32, 1, None, 0, 0.1, P, big, None),
               cdll.mi355_cache_evict(c, 10, 5, P * 16, P, big, None)):
        assert rc in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED)
        assert cdll.mi355_last_error()
    assert cdll.mi355_fmha_paged(None, P, P, P, 32, 1, None, 0.1, P, big, None) == lib.ERR_BAD_ARGUMENT


def test_attention_refuses_bad_arguments(lib):
    cdll, c, big = lib.load(), cache(lib), 1 << 60

    def call(Q=P, O=P, Hq=32, S=1, strides=None, scale=0.1, ws=P, size=big):
        st = None if strides is None else (ctypes.c_int64 * 6)(*strides)
        return cdll.mi355_fmha_paged(c, Q, O, P, Hq, S, st, scale, ws, size, None)

    ok = [4096, 128, 128, 4096, 128, 128]
    for kw in (dict(Q=None), dict(O=None), dict(Q=P + 2), dict(O=P + 2), dict(Hq=0), dict(Hq=31), dict(S=0), dict(scale=0.0), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(S=16384), dict(strides=[-8] + ok[1:]), dict(strides=[4] + ok[1:]), dict(strides=ok[:2] + [1 << 24] + ok[3:]),
               dict(strides=ok[:4] + [64, 128]), dict(strides=ok[:3] + [0, 128, 128])):
        assert call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw
    # launches of more workgroups than there may be
    many = cache(lib, B=8000, table_stride=8)
    assert cdll.mi355_fmha_paged(many, P, P, P, 32, 100, None, 0.1, P, big, None) == lib.ERR_UNSUPPORTED
    far = cache(lib, max_pages=1 << 20, table_stride=1 << 20)
    assert cdll.mi355_fmha_key_weights(far, P, P, 32, 16383, None, 0, 0.1, P, big, None) == lib.ERR_UNSUPPORTED
    # a workspace is needed for the scores that the account is made from
    need = cdll.mi355_fmha_paged_workspace_bytes(c, 32, 1, 1)
    assert need > 0
    for kw in (dict(ws=None), dict(size=need - 1), dict(ws=P + 4)):
        assert call(**kw) == lib.ERR_BAD_ARGUMENT
        assert b"workspace" in cdll.mi355_last_error()
    # none without an account, up to 512 keys
    assert cdll.mi355_fmha_paged_workspace_bytes(cache(lib, weights=None), 32, 1, 1) == 0


def test_workspaces_of_refused_calls_are_zero_bytes(lib):
    """Sizes whose products leave the range of an int, or are zero in it, among them."""
    cdll = lib.load()
    sizes = [dict(page_size=1 << 16, max_pages=1 << 16), dict(page_size=1 << 30, max_pages=4), dict(max_pages=(1 << 24) + 1), dict(B=1 << 16, Hkv=1 << 16), dict(page_size=24),
             dict(page_size=0), dict(B=0)]
    for bad in sizes:
        c = cache(lib, **bad)
        assert cdll.mi355_fmha_paged_workspace_bytes(c, 1 << 16, 4, 1) == 0
        assert cdll.mi355_fmha_key_weights_workspace_bytes(c, 1 << 16, 4, 0) == 0
        assert cdll.mi355_cache_evict_workspace_bytes(c, 32) == 0
    for Hq, S in ((1 << 16, 1 << 16), (1 << 16, 1 << 15), (1 << 20, 1 << 30), (8, 1 << 16), (7, 4), (8, 0), (0, 4)):
        for weights in (None, P):
            c = cache(lib, weights=weights)
            assert cdll.mi355_fmha_paged_workspace_bytes(c, Hq, S, 1) == 0
            assert cdll.mi355_fmha_key_weights_workspace_bytes(c, Hq, S, 0) == 0
    assert cdll.mi355_cache_evict_workspace_bytes(cache(lib), 0) == 0


def test_an_account_of_more_rows_than_a_launch_takes_is_refused(lib):
    cdll, big = lib.load(), 1 << 60
    wide = dict(B=1, Hkv=1, max_pages=1 << 20, table_stride=1 << 20)   # 65536 blocks of keys, 16 tiles of rows a workgroup
    assert cdll.mi355_fmha_paged(cache(lib, **wide), P, P, P, 4, 16000, None, 0.1, P, 0, None) == lib.ERR_BAD_ARGUMENT   # (no workspace: sizes are fine)
    assert cdll.mi355_fmha_paged(cache(lib, **wide), P, P, P, 32768, 1, None, 0.1, P, big, None) == lib.ERR_UNSUPPORTED
    assert b"more than a call takes" in cdll.mi355_last_error()


def test_prompts_of_many_heads_and_tokens_are_taken(lib):
    """The workspaces of calls of 65536 query columns a kv head and more are sized, and only a missing one is refused."""
    cdll = lib.load()
    for Hq, Hkv, S, last, pages in ((64, 8, 8192, 0, 512), (32, 8, 16384, 0, 1024), (32, 1, 2048, 0, 128), (64, 8, 8192, 64, 512), (32, 8, 1 << 20, 5, 1 << 16)):
        c = cache(lib, B=1, Hkv=Hkv, max_pages=pages, table_stride=pages)
        if last == 0:
            need = cdll.mi355_fmha_paged_workspace_bytes(c, Hq, S, 1)
            assert 0 < need < 1 << 32
            assert cdll.mi355_fmha_paged(c, P, P, P, Hq, S, None, 0.1, None, need, None) == lib.ERR_BAD_ARGUMENT and b"workspace" in cdll.mi355_last_error()
        need = cdll.mi355_fmha_key_weights_workspace_bytes(c, Hq, S, last)
        assert (need > 0 or last > 0) and need < 1 << 32
        if need:
            assert cdll.mi355_fmha_key_weights(c, P, P, Hq, S, None, last, 0.1, None, need, None) == lib.ERR_BAD_ARGUMENT and b"workspace" in cdll.mi355_last_error()
    # more rows than a sequence has keys, more columns than there may be
    for Hq, S, last in ((64, 8193, 0), (8, 1 << 16, 0), (8, (1 << 28) + 1, 1)):
        c = cache(lib, B=1, Hkv=8, max_pages=512, table_stride=512)
        assert cdll.mi355_fmha_key_weights(c, P, P, Hq, S, None, last, 0.1, P, 1 << 60, None) == lib.ERR_UNSUPPORTED
        assert cdll.mi355_fmha_key_weights_workspace_bytes(c, Hq, S, last) == 0


def test_a_scale_that_is_infinite_in_powers_of_two_is_refused(lib):
    """The kernels take exponentials to the base 2, of scores times scale * log2 e."""
    cdll, c = lib.load(), cache(lib)
    for scale, word in ((2.4e38, b"scale"), (3.0e38, b"scale"), (2.2e38, b"workspace"), (1e-45, b"workspace")):
        assert cdll.mi355_fmha_paged(c, P, P, P, 32, 1, None, scale, None, 0, None) == lib.ERR_BAD_ARGUMENT and word in cdll.mi355_last_error()
        need = cdll.mi355_fmha_key_weights_workspace_bytes(c, 32, 1000, 0)
        assert need > 0
        assert cdll.mi355_fmha_key_weights(c, P, P, 32, 1000, None, 0, scale, None, 0, None) == lib.ERR_BAD_ARGUMENT and word in cdll.mi355_last_error()


def test_the_other_entry_points_refuse_bad_arguments(lib):
    cdll, c, big = lib.load(), cache(lib), 1 << 60
    row = 48 * 128

    def rope(qkv=P, S=2, q_heads=32, x_batch=2 * row, x_row=row, cos=P, sin=P, pos=P, pos_batch=0, n=100):
        return cdll.mi355_rope_paged(c, qkv, S, q_heads, 0, x_batch, x_row, cos, sin, pos, pos_batch, n, None)

    for kw in (dict(qkv=None), dict(cos=None), dict(sin=None), dict(pos=None), dict(qkv=P + 2), dict(cos=P + 4), dict(S=0), dict(q_heads=-1), dict(n=0),
               dict(x_row=row - 8), dict(x_row=row + 4), dict(x_batch=row - 8), dict(x_batch=-8), dict(pos_batch=1), dict(S=1 << 30), dict(S=1 << 22)):
        assert rope(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw

    def kw_call(Q=P, LSE=P, Hq=32, S=4, strides=None, last=0, scale=0.1, cc=c):
        st = None if strides is None else (ctypes.c_int64 * 3)(*strides)
        return cdll.mi355_fmha_key_weights(cc, Q, LSE, Hq, S, st, last, scale, P, big, None)

    for kw in (dict(Q=None), dict(LSE=None), dict(Hq=31), dict(S=0), dict(last=-1), dict(scale=-1.0), dict(strides=[8, 8, 4]), dict(cc=cache(lib, weights=None))):
        assert kw_call(**kw) in (lib.ERR_BAD_ARGUMENT, lib.ERR_UNSUPPORTED), kw

    def evict(budget=10, recent=5, out=P * 16, ws=P, size=big, cc=c):
        return cdll.mi355_cache_evict(cc, budget, recent, out, ws, size, None)

    need = cdll.mi355_cache_evict_workspace_bytes(c, 10)
    for kw in (dict(budget=0), dict(recent=-1), dict(out=None), dict(out=P), dict(out=P + 12), dict(out=P - 12), dict(ws=None), dict(size=need - 1),
               dict(cc=cache(lib, weights=None)), dict(cc=cache(lib, key_positions=None))):
        assert evict(**kw) == lib.ERR_BAD_ARGUMENT, kw


def tensors(B=2, Hq=8, Hkv=2, S=1, page=16, n_pages=5, max_pages=2):
    kv = torch.zeros(n_pages, 2 * Hkv, page, 128, dtype=torch.float16)
    table, lens = torch.zeros(B, max_pages, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    return dict(q=torch.zeros(B, Hq, S, 128, dtype=torch.float16), kv_pages=kv, block_table=table, seq_lens=lens)


def test_operators_refuse_what_is_not_on_the_gpu_and_wrong_shapes():
    t = tensors()
    w, pos = torch.zeros(5, 2, 16), torch.zeros(5, 2, 16, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.fine_fmha_paged(**t)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.fine_evict_paged(t["kv_pages"], t["block_table"], t["seq_lens"], w, pos, 4, 2)
    for name, bad in (("kv_pages", torch.zeros(5, 3, 16, 128, dtype=torch.float16)), ("kv_pages", torch.zeros(5, 4, 16, 64, dtype=torch.float16)),
                      ("kv_pages", torch.zeros(5, 4, 16, 128)), ("kv_pages", torch.zeros(0, 4, 16, 128, dtype=torch.float16)),
                      ("kv_pages", torch.zeros(5, 4, 128, 16, dtype=torch.float16).transpose(2, 3)), ("block_table", torch.zeros(2, dtype=torch.int32)),
                      ("block_table", torch.zeros(2, 0, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match=name):
            ops.fine_fmha_paged(**dict(t, **{name: bad}))


def test_operators_name_what_they_write():
    for name, written in (("finefmha_paged", ["weights"]), ("finefmha_paged_lse", ["weights"]), ("rope_paged", ["qkv", "kv_pages", "weights", "key_positions"]),
                          ("key_weights", ["weights"]), ("evict_paged", ["kv_pages", "weights", "key_positions"])):
        schema = getattr(torch.ops.fmha_unified, name).default._schema
        assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == written


class Seen(TorchDispatchMode):
    """Names of the operators that torch's dispatcher is asked for; none of them runs."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return tuple(torch.zeros(1) for _ in func._schema.returns) if len(func._schema.returns) > 1 else torch.zeros(1) if func._schema.returns else None


def test_what_watches_the_dispatcher_sees_the_functions():
    t, one = tensors(), torch.ones(50, 64)
    w, pos, p = torch.zeros(5, 2, 16), torch.zeros(5, 2, 16, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pool = (t["kv_pages"], t["block_table"], t["seq_lens"])
    qkv, lse = torch.zeros(2, 1, 12, 128, dtype=torch.float16), torch.zeros(2, 8, 1)
    with Seen() as seen:
        ops.fine_fmha_paged(**t)
        ops.fine_fmha_paged_with_lse(**t, weights=w)
        ops.fine_rope_paged(qkv, *pool, one, one, p, 8, key_positions=pos)
        ops.fine_key_weights(t["q"], lse, *pool, w)
        ops.fine_evict_paged(*pool, w, pos, 4, 2)
    assert seen.names == ["fmha_unified::" + n for n in ("finefmha_paged", "finefmha_paged_lse", "rope_paged", "key_weights", "evict_paged")]


def test_a_cache_hands_out_pages_and_takes_them_back():
    from llama_layer import FinePagedKVCache
    c = FinePagedKVCache(3, 10, 2, page_size=16, max_pages=4, device="cpu", account=True)

    def consistent():
        used = [p for row in c._pages for p in row]
        assert len(set(used)) == len(used) and sorted(used + c._free) == list(range(10))
        for b, row in enumerate(c._pages):
            assert c.block_table[b].tolist() == row + [-1] * (4 - len(row)) and len(row) == -(-c.lengths[b] // 16)
        assert c.seq_lens.tolist() == c.lengths and c.next_positions.tolist() == c.positions

    c.extend([20, 0, 33])
    consistent()
    assert c.lengths == [20, 0, 33] and c.free_pages == 5
    for new in ([0, 65, 0], [16, 64, 16], [1, 2], [-1, 0, 0]):      # a sequence, the pool, another batch, fewer than none
        with pytest.raises(ValueError):
            c.extend(new)
        consistent()
        assert c.lengths == [20, 0, 33]
    c.extend([12, 1, 15])
    consistent()
    c.take_back([12, 1, 2])
    consistent()
    assert c.lengths == [20, 0, 46]
    with pytest.raises(ValueError):
        c.take_back([0, 1, 0])
    c.release(2)
    consistent()
    assert c.lengths == [20, 0, 0] and c.positions == [20, 0, 0]
    c.extend([1, 1, 1])
    consistent()
    with pytest.raises(ValueError, match="account"):
        FinePagedKVCache(1, 4, 1, device="cpu").evict(3, 1)


def test_calls_get_the_columns_in_use():
    from llama_layer import FinePagedKVCache
    c = FinePagedKVCache(2, 100, 1, page_size=48, device="cpu")          # steps of 6 pages, 288 keys
    for new, rows, width in (([0, 0], 1, 6), ([288, 5], 5, 6), ([1, 0], 1, 12), ([0, 0], 2000, 42), ([0, 0], 1 << 20, 100)):
        c.extend(new)
        table = c.table_in_use(rows)
        assert table.shape == (2, width) and table.data_ptr() == c.block_table.data_ptr() and table.stride(0) == 100
    assert FinePagedKVCache(1, 4, 1, page_size=512, device="cpu").table_in_use().shape == (1, 1)


def test_positions_of_a_cache_follow_those_that_were_given():
    from llama_layer import FinePagedKVCache
    c = FinePagedKVCache(3, 20, 1, page_size=16, device="cpu")
    ids = lambda *rows: torch.tensor(rows, dtype=torch.int32)
    for new, given, want in (([2, 2, 2], None, [2, 2, 2]), ([2, 2, 2], ids([7, 8], [90, 91], [4, 5]), [9, 92, 6]), ([1, 1, 1], None, [10, 93, 7]),
                             ([0, 2, 1], ids([50, 51], [60, 61], [70, 71]), [10, 62, 71]), ([0, 0, 0], ids([1], [1], [1]), [10, 62, 71]),
                             ([1, 0, 2], ids([30, 31]), [31, 62, 32]), ([3, 3, 3], ids([40, 41, 42]), [43, 43, 43])):
        c.extend(new)
        if given is not None:
            c.went_to(given, new)
        assert c.positions == want and c.next_positions.tolist() == want
    c.went_to(ids([40, 41, 52]), [3, 3, 3])
    c.take_back([1, 0, 3])
    c.extend([0, 2, 0])
    c.release(0)
    assert c.positions == [0, 55, 50] and c.next_positions.tolist() == [0, 55, 50]
    c.release(1)
    assert c.positions == [0, 0, 50]
