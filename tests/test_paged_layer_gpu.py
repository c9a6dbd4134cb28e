"""The decoder layer over a cache in pages: against the oracle's layer sequence by sequence, and with eviction against attention over what is kept."""
import pytest
import torch

import serving_oracle as so
from llama_layer import FineKVCache, FineLlamaDecoderLayer, FinePagedKVCache

pytestmark = pytest.mark.gpu


def layer_weights(H, n_q, n_kv, F, seed=0):
    g = lambda shape, s, std: so.randn_fp16(shape, seed + s, std)
    w = dict(q=g((n_q * 128, H), 1, 0.03), k=g((n_kv * 128, H), 2, 0.03), v=g((n_kv * 128, H), 3, 0.03), o=g((H, n_q * 128), 4, 0.03),
             gate=g((F, H), 5, 0.03), up=g((F, H), 6, 0.03), down=g((H, F), 7, 0.03))
    w["ln1"] = (1 + 0.1 * g((H,), 8, 1.0).float()).half()
    w["ln2"] = (1 + 0.1 * g((H,), 9, 1.0).float()).half()
    return w


def layer_close(out, ref):
    # the layer's tolerance everywhere: its stages are rounded to fp16 one after the other
    out, ref = out.float().cpu(), ref.float()
    rel, worst = float((out - ref).norm() / ref.norm()), float((out - ref).abs().max() / ref.abs().max())
    assert rel <= 2e-3 and worst <= 2e-2, (rel, worst)


def keys_of(cache, b):
    j = torch.arange(cache.lengths[b], device=cache.kv_pages.device)
    page = cache.kv_pages.shape[2]
    return cache.kv_pages[cache.block_table[b].long()[j // page], :, j % page].transpose(0, 1).float().cpu()    # [2 n_kv, n, 128]


@pytest.mark.parametrize("account", [False, True])
@pytest.mark.parametrize("lens,steps", [([300, 57, 1], 3), ([40], 2)])
def test_layer_over_pages_is_the_oracles(gpu, lens, steps, account):
    H, n_q, n_kv, F, B, S = 512, 8, 2, 1024, len(lens), max(lens)
    w = layer_weights(H, n_q, n_kv, F, seed=20)
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in w.items()}, n_q, n_kv, max_positions=1024)
    cache = FinePagedKVCache(B, 40, n_kv, page_size=16, max_pages=22, device=gpu, account=account)
    x = so.randn_fp16((B, S, H), 1)
    out = layer(x.to(gpu), kv_cache=cache, new_lens=lens, time_attention=True)
    refs = []
    for b, n in enumerate(lens):
        ref, k, v = so.llama_decoder_layer_ref(x[b:b + 1, :n], w, torch.arange(n)[None], n_q, n_kv)
        layer_close(out[b:b + 1, :n], ref)
        refs.append((k, v))
    assert cache.lengths == list(lens)
    for t in range(steps):
        S = 1 if t < steps - 1 else 3                     # the last call brings three drafted tokens
        xt = so.randn_fp16((B, S, H), 100 + t)
        out = layer(xt.to(gpu), kv_cache=cache, time_attention=True)
        for b in range(B):
            n = cache.lengths[b] - S
            ref, k, v = so.llama_decoder_layer_ref(xt[b:b + 1], w, torch.arange(n, n + S)[None], n_q, n_kv, past_k=refs[b][0], past_v=refs[b][1])
            layer_close(out[b:b + 1], ref)
            refs[b] = (k, v)
            got = keys_of(cache, b)
            assert (got[:n_kv] - k[0]).abs().max() <= 2e-2 and (got[n_kv:] - v[0]).abs().max() <= 2e-2
    assert len(layer.attn_ms["prefill"]) == 2 and len(layer.attn_ms["decode"]) == steps - 1
    if account:
        # every query of every head spreads a weight of one over the keys it sees (fp16: its log-sum-exp is half a step off at most)
        for b in range(B):
            j = torch.arange(cache.lengths[b], device=gpu)
            where = cache.block_table[b].long()[j // 16]
            total = cache.weights[where, :, j % 16].double().sum(0)
            queries = (n_q // n_kv) * cache.lengths[b]
            assert (total - queries).abs().max() <= queries * (2.0 ** -11 + 2.0 ** -16)
            assert (cache.key_positions[where, :, j % 16] == j[:, None]).all()


def test_layer_over_pages_and_over_a_contiguous_cache(gpu):
    """The same tokens through both caches, whose kernels round alike (half a step of an intermediate here and there)."""
    H, n_q, n_kv, F, B = 512, 4, 2, 1024, 2
    w = layer_weights(H, n_q, n_kv, F, seed=50)
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in w.items()}, n_q, n_kv, max_positions=256)
    paged, fine = FinePagedKVCache(B, 30, n_kv, page_size=48, device=gpu), FineKVCache(B, 200, n_kv, device=gpu)
    for t, S in enumerate((70, 1, 40, 1)):                 # the third brings a chunk of a prompt over what is there
        x = so.randn_fp16((B, S, H), 60 + t).to(gpu)
        layer_close(layer(x, kv_cache=paged), layer(x, kv_cache=fine).float().cpu())
        assert paged.lengths == [fine.length] * B
    for b in range(B):
        assert (keys_of(paged, b) - fine.kv[b, :, :fine.length].float().cpu()).abs().max() <= 2e-2


def test_steps_with_eviction_attend_to_what_is_kept(gpu):
    H, n_q, n_kv, F, B, budget = 512, 8, 2, 1024, 2, 64
    w = layer_weights(H, n_q, n_kv, F, seed=70)
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in w.items()}, n_q, n_kv, max_positions=512)
    cache = FinePagedKVCache(B, 24, n_kv, page_size=16, max_pages=12, device=gpu, account=True)
    x = so.randn_fp16((B, 130, H), 1)
    layer(x.to(gpu), kv_cache=cache, new_lens=[130, 50])
    assert cache.free_pages == 24 - 9 - 4
    cache.evict(budget, 20)
    assert cache.lengths == [64, 50] and cache.positions == [130, 50] and cache.free_pages == 24 - 4 - 4
    for t in range(20):
        xt = so.randn_fp16((B, 1, H), 200 + t)
        kept = [keys_of(cache, b) for b in range(B)]
        at = list(cache.positions)
        out = layer(xt.to(gpu), kv_cache=cache)
        for b in range(B):
            ref, _, _ = so.llama_decoder_layer_ref(xt[b:b + 1], w, torch.tensor([[at[b]]]), n_q, n_kv, past_k=kept[b][None, :n_kv], past_v=kept[b][None, n_kv:])
            layer_close(out[b:b + 1], ref)
        if t % 4 == 3:
            cache.evict(budget, 20)
            assert max(cache.lengths) <= budget and cache.seq_lens.tolist() == cache.lengths
            # the newest tokens are among the kept ones
            for b in range(B):
                j = torch.arange(cache.lengths[b], device=gpu)
                where = cache.key_positions[cache.block_table[b].long()[j // 16], :, j % 16]
                for h in range(n_kv):
                    assert set(range(max(0, cache.positions[b] - 20), cache.positions[b])) <= set(where[:, h].tolist())
    assert cache.positions == [150, 70] and cache.lengths == [64, 64]
    with pytest.raises(ValueError):
        cache.take_back([1, 0])                       # cut a moment ago: the last slot is not the last token
    layer(so.randn_fp16((B, 3, H), 300).to(gpu), kv_cache=cache)
    with pytest.raises(ValueError):
        cache.take_back([4, 0])
    cache.take_back([2, 3])
    assert cache.lengths == [65, 64] and cache.positions == [151, 70] and cache.seq_lens.tolist() == [65, 64]


def test_a_long_prompt_of_many_heads_with_an_account(gpu):
    """8192 tokens of 64 query heads on 8 kv heads, as without an account; each row spreads a weight of one a head."""
    H, n_q, n_kv, F, S = 512, 64, 8, 1024, 8192
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in layer_weights(H, n_q, n_kv, F, seed=90).items()}, n_q, n_kv, max_positions=S)
    x = so.randn_fp16((1, S, H), 5).to(gpu)
    caches = [FinePagedKVCache(1, S // 64, n_kv, page_size=64, device=gpu, account=account) for account in (False, True)]
    plain, counted = [layer(x, kv_cache=c) for c in caches]
    assert torch.equal(plain, counted)
    cache = caches[1]
    total = cache.weights[cache.block_table[0].long()].double().sum((0, 2))
    assert ((total - 8 * S).abs() <= 8 * S * (2.0 ** -11 + 2.0 ** -16)).all()


def test_calls_cost_what_is_in_use_whatever_the_pool(gpu):
    """A table as wide as a large pool: the workspaces of a step, a chunk of a prompt and an eviction do not grow with it, results are those of a narrow one."""
    H, n_q, n_kv, F, B = 512, 8, 2, 1024, 8
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in layer_weights(H, n_q, n_kv, F, seed=30).items()}, n_q, n_kv, max_positions=512)
    wide, narrow = FinePagedKVCache(B, 20000, n_kv, page_size=16, device=gpu, account=True), FinePagedKVCache(B, 200, n_kv, page_size=16, max_pages=64, device=gpu, account=True)
    lens = [120, 50, 33, 1, 0, 99, 16, 17]

    def both(call):
        results = []
        for cache in (wide, narrow):
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            results.append(call(cache))
            torch.cuda.synchronize()
            assert torch.cuda.max_memory_allocated() - before <= 64 << 20
        return results

    for S, new in ((120, lens), (1, None), (20, [20] * 7 + [3]), (1, None)):
        x = so.randn_fp16((B, S, H), 40 + S).to(gpu)
        a, b = both(lambda cache: layer(x, kv_cache=cache, new_lens=new))
        assert torch.equal(a, b)
    both(lambda cache: cache.evict(60, 20))
    assert wide.lengths == narrow.lengths and wide.seq_lens.tolist() == wide.lengths
    for b in range(B):
        assert torch.equal(keys_of(wide, b), keys_of(narrow, b))
    x = so.randn_fp16((B, 1, H), 9).to(gpu)
    a, b = both(lambda cache: layer(x, kv_cache=cache))
    assert torch.equal(a, b)


def test_positions_go_on_behind_those_that_were_given(gpu):
    H, n_q, n_kv, F, B = 512, 4, 2, 1024, 2
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in layer_weights(H, n_q, n_kv, F, seed=11).items()}, n_q, n_kv, max_positions=1200)
    make = lambda: FinePagedKVCache(B, 40, n_kv, page_size=16, device=gpu, account=True)
    given, mixed = make(), make()
    x = so.randn_fp16((B, 100, H), 1).to(gpu)
    first = torch.stack((torch.arange(1000, 1100), torch.arange(500, 600))).to(gpu)
    new = [100, 60]
    for cache in (given, mixed):
        layer(x, first, kv_cache=cache, new_lens=new)
        assert cache.positions == [1100, 560] and cache.next_positions.tolist() == [1100, 560]
        cache.evict(50, 20)
        assert cache.positions == [1100, 560]
    for t in range(8):
        xt = so.randn_fp16((B, 1, H), 20 + t).to(gpu)
        a = layer(xt, torch.tensor([[1100 + t], [560 + t]], device=gpu), kv_cache=given)
        b = layer(xt, kv_cache=mixed)
        assert torch.equal(a, b)
    for cache in (given, mixed):
        assert cache.positions == [1108, 568] and cache.next_positions.tolist() == [1108, 568]
        cache.evict(50, 20)
        for b in range(B):                             # the newest tokens are the last of the text
            j = torch.arange(50, device=gpu)
            where = cache.key_positions[cache.block_table[b].long()[j // 16], :, j % 16]
            for h in range(n_kv):
                assert set(range(cache.positions[b] - 20, cache.positions[b])) <= set(where[:, h].tolist())
    # one row of positions for all sequences; sequences without a token stay where they are
    layer(so.randn_fp16((B, 3, H), 50).to(gpu), torch.arange(1150, 1153)[None].to(gpu), kv_cache=mixed, new_lens=[0, 2])
    assert mixed.positions == [1108, 1152]
    mixed.take_back([0, 1])
    assert mixed.positions == [1108, 1151] and mixed.next_positions.tolist() == [1108, 1151]
    with pytest.raises(ValueError, match="max_positions"):
        layer(so.randn_fp16((B, 50, H), 51).to(gpu), kv_cache=mixed)
    mixed.release(0)
    assert mixed.positions == [0, 1151]


def test_a_subclass_of_the_cache_is_one(gpu):
    class Mine(FinePagedKVCache):
        pass

    H, n_q, n_kv, F = 512, 4, 2, 1024
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in layer_weights(H, n_q, n_kv, F).items()}, n_q, n_kv, max_positions=64)
    x = so.randn_fp16((2, 20, H), 3).to(gpu)
    a, b = [layer(x, kv_cache=kind(2, 6, n_kv, page_size=16, device=gpu), new_lens=[20, 7]) for kind in (FinePagedKVCache, Mine)]
    assert torch.equal(a[0], b[0]) and torch.equal(a[1, :7], b[1, :7])


def test_layer_over_pages_refuses(gpu):
    H, n_q, n_kv, F = 512, 4, 2, 1024
    layer = FineLlamaDecoderLayer({k: v.to(gpu) for k, v in layer_weights(H, n_q, n_kv, F).items()}, n_q, n_kv, max_positions=64)
    cache = FinePagedKVCache(2, 6, n_kv, page_size=16, device=gpu)
    x = torch.zeros(2, 20, H, dtype=torch.float16, device=gpu)
    for bad, kw in ((x[:1], {}), (x, {"new_lens": [20]}), (x, {"new_lens": [21, 1]}), (torch.zeros(2, 65, H, dtype=torch.float16, device=gpu), {})):
        with pytest.raises(ValueError):
            layer(bad, kv_cache=cache, **kw)
        assert cache.lengths == [0, 0] and cache.free_pages == 6
    with pytest.raises(RuntimeError):
        layer(x.bfloat16(), kv_cache=cache)          # not the weights' type: nothing was filed
    assert cache.lengths == [0, 0] and cache.free_pages == 6 and cache.seq_lens.tolist() == [0, 0]
    layer(x, kv_cache=cache)
    with pytest.raises(ValueError):
        layer(torch.zeros(2, 40, H, dtype=torch.float16, device=gpu), kv_cache=cache)     # no pages left
    assert cache.lengths == [20, 20]
    with pytest.raises(ValueError):
        layer(x, kv_cache=FineKVCache(2, 64, n_kv, device=gpu), new_lens=[20, 20])
