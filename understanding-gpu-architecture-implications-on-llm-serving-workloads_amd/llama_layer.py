"""A Llama decoder layer on the MI355X kernels: the in-model caller of fine_fmha, rebuilt without its copies.

The reference measures its attention kernels inside a patched Hugging Face layer
(benchmarks/flashattn-cuda/modeling_llama.py): LlamaSdpaAttention.forward (:652-704) projects with three nn.Linear
calls, transposes to [B, H, S, D], applies RoPE, expands K/V with repeat_kv (:670-671), calls
``fmha_unified.ops.fine_fmha`` (:687-690), transposes back with a copy (:700) and projects; LlamaDecoderLayer.forward
(:755-781) wraps it in RMSNorm, residual adds and the gate/up/down MLP (:227), all as separate PyTorch kernels.

Here one layer is eight launches, with or without a KV cache, prefill and generation step alike (one more where
the gate/up epilogue does not apply, an MLP width that is no multiple of 32, and SiLU*up runs on its own), with no layout copies:
    rmsnorm -> QKV GEMM (one fused NT GEMM on the nn.Linear weights) -> RoPE in place on the q and k heads of the
    projection (k goes straight into the KV cache when there is one) -> attention reading q, k, v where they lie
    (strided operands, GQA inside the kernel, output written as [B, S, Hq*D]) -> O projection with the residual
    added in its epilogue -> rmsnorm -> gate/up GEMM with SiLU(gate)*up applied in its epilogue -> down GEMM with the
    residual added in its epilogue.
With up to 8 rows (a generation step) RoPE is part of the QKV product, and each norm of the product behind it where that pays (1 or 2 rows
up to 7680 wide, 4 up to 4608, 8 up to 2560, fewer in front of a wide MLP: `norm_fits` in csrc/hgemm.hip): five to seven launches.
With a cache in pages (FinePagedKVCache: sequences of different lengths) norm, QKV product and rotary embedding with filing are three launches; the
attention is over the pages, or for a prompt over its projection, and what the keys were attended to is kept where eviction will ask for it.
Weights keep the nn.Linear layout ([out_features, in_features]); nothing is transposed or repacked beyond
concatenating q/k/v and interleaving gate/up along the output dimension once at construction.
"""
import torch

import mi355_serving as lib
from fmha_unified.ops import fine_evict_paged
from mi355_serving import _C

__all__ = ["FineKVCache", "FinePagedKVCache", "FineLlamaDecoderLayer", "rope_tables"]


def rope_tables(n_positions, head_dim=128, base=10000.0, device="cuda"):
    """cos, sin [n_positions, head_dim / 2] fp32 (LlamaRotaryEmbedding, modeling_llama.py:113,119-132)."""
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.int64).float() / head_dim))
    ang = torch.arange(n_positions, dtype=torch.float32)[:, None] * inv_freq[None, :]
    return ang.cos().contiguous().to(device), ang.sin().contiguous().to(device)


class FineKVCache:
    """Static key/value cache of one layer: one tensor [B, 2 * n_kv, max_len, 128], head-major (the keys of a (sequence, head)
    are one contiguous stream for the generation-step attention, which reads them from HBM 3 us faster at batch 8 over 8192
    keys than 256-byte pieces 4 KiB apart), key heads followed by value heads, so one kernel launch files both. `k` and
    `v` are [B, max_len, n_kv, 128] views of it that the attention kernel reads in place; `rows(past, S)` is the
    [B, S, 2 * n_kv, 128] view of S new tokens."""

    def __init__(self, batch, max_len, n_kv, head_dim=128, device="cuda", dtype=torch.float16):
        self.kv = torch.empty((batch, 2 * n_kv, max_len, head_dim), dtype=dtype, device=device)
        self.k = self.kv[:, :n_kv].transpose(1, 2)
        self.v = self.kv[:, n_kv:].transpose(1, 2)
        self.length = 0

    @property
    def max_len(self):
        return self.kv.shape[2]

    def rows(self, past, S):
        return self.kv[:, :, past:past + S].transpose(1, 2)


class FinePagedKVCache:
    """Key/value cache of one layer in pages, for sequences of different lengths that come and go: a pool `kv_pages` [n_pages, 2 * n_kv,
    page_size, 128], of which each of `batch` sequences owns the pages in its row of `block_table` [batch, max_pages]. `seq_lens` and
    `next_positions` (int32, on the device) hold each sequence's keys and the position of its next token, one behind its last; `lengths` and
    `positions` are the same on the host, which hands out the pages (`positions` waits for the device once after a call with position_ids of its
    own). With `account`, `weights` and `key_positions` [n_pages, n_kv, page_size] keep what `evict` goes by: the attention that each key has
    had, the position of its token.

    The layer's forward makes room with `extend` and files its tokens; `evict` cuts long sequences, `release` frees one."""

    def __init__(self, batch, n_pages, n_kv, page_size=32, max_pages=None, head_dim=128, device="cuda", dtype=torch.float16, account=False):
        max_pages = n_pages if max_pages is None else max_pages
        self.kv_pages = torch.zeros((n_pages, 2 * n_kv, page_size, head_dim), dtype=dtype, device=device)
        self.block_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.next_positions = torch.zeros(batch, dtype=torch.int32, device=device)
        self.weights = torch.zeros((n_pages, n_kv, page_size), device=device) if account else None
        self.key_positions = torch.zeros((n_pages, n_kv, page_size), dtype=torch.int32, device=device) if account else None
        self.lengths, self._positions = [0] * batch, [0] * batch   # (positions: None where the device alone knows them)
        self._in_order = [0] * batch      # tokens at the end of each sequence that no eviction has moved
        self._pages = [[] for _ in range(batch)]
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    @property
    def positions(self):
        if self._positions is None:
            self._positions = self.next_positions.tolist()
        return self._positions

    @positions.setter
    def positions(self, positions):
        self._positions = positions

    def went_to(self, position_ids, new):
        """The last new[b] tokens of each sequence, which `extend` made room for, are those at position_ids [1 or batch, new or more] (int32, on the
        device): positions go on behind them."""
        came = [b for b, n in enumerate(new) if n > 0]
        if not came:
            return
        if len(came) == len(new) and min(new) == max(new):
            self.next_positions.copy_(position_ids[:, new[0] - 1] + 1)
        else:
            index = torch.tensor([came, [b if position_ids.shape[0] > 1 else 0 for b in came], [new[b] - 1 for b in came]], device=position_ids.device)
            self.next_positions[index[0]] = position_ids[index[1], index[2]] + 1
        self._positions = None

    def table_in_use(self, rows=0):
        """The columns of the block table that the longest sequence needs, or one of `rows` keys, in steps of 256 keys: launches, workspaces and the choice
        of kernels go by the width of the table that a call is given, and the pool's may be a thousand times what is in use. (A call that is captured keeps
        its table: one that is replayed as the lengths go on needs as many columns as they will.)"""
        page = self.kv_pages.shape[2]
        step = -(-256 // page)
        return self.block_table[:, :-(-max(rows, 1, *self.lengths) // (step * page)) * step]

    def extend(self, new):
        """Room for new[b] more tokens of each sequence, whose lengths and positions go on by that many. ValueError, and nothing changed, where the
        pool or the table has no more."""
        page, width = self.kv_pages.shape[2], self.block_table.shape[1]
        if len(new) != len(self.lengths) or any(n < 0 for n in new):
            raise ValueError("new tokens of %d sequences expected, got %r" % (len(self.lengths), new))
        lengths = [n + more for n, more in zip(self.lengths, new)]
        wanted = [max(0, -(-n // page) - len(have)) for n, have in zip(lengths, self._pages)]
        if sum(wanted) > len(self._free) or any(n > width * page for n in lengths):
            raise ValueError("a cache of %d free pages of %d tokens, %d a sequence, cannot take %r more after %r" %
                             (len(self._free), page, width, list(new), self.lengths))
        for b, more in enumerate(wanted):
            for _ in range(more):
                self._pages[b].append(self._free.pop())
        if any(wanted):
            self._write_table([b for b, more in enumerate(wanted) if more])
        self.lengths = lengths
        if self._positions is not None:
            self._positions = [n + more for n, more in zip(self._positions, new)]
        self._in_order = [n + more for n, more in zip(self._in_order, new)]
        step = new[0] if all(n == new[0] for n in new) else torch.tensor(new, dtype=torch.int32, device=self.seq_lens.device)
        self.seq_lens += step
        self.next_positions += step

    def take_back(self, new):
        """The last new[b] tokens of each sequence are no longer its own (a call that failed; drafted tokens that were not accepted); ValueError for more
        than have come since it was cut, which leaves no order. Positions go back by as many. The account of the others keeps what those added to it."""
        if len(new) != len(self.lengths) or any(not 0 <= n <= have for n, have in zip(new, self._in_order)):
            raise ValueError("cannot take %r tokens back where %r have come" % (new, self._in_order))
        self._in_order = [n - less for n, less in zip(self._in_order, new)]
        self.lengths = [n - less for n, less in zip(self.lengths, new)]
        if self._positions is not None:
            self._positions = [n - less for n, less in zip(self._positions, new)]
        step = new[0] if all(n == new[0] for n in new) else torch.tensor(new, dtype=torch.int32, device=self.seq_lens.device)
        self.seq_lens -= step
        self.next_positions -= step
        self._give_back(range(len(new)))

    def evict(self, budget, recent):
        """Cuts every sequence longer than `budget` to it (fmha_unified.ops.fine_evict_paged) and frees the pages behind it."""
        if self.weights is None:
            raise ValueError("eviction needs a cache made with account=True")
        if all(n <= budget for n in self.lengths):
            return
        self.seq_lens.copy_(fine_evict_paged(self.kv_pages, self.table_in_use(), self.seq_lens, self.weights, self.key_positions, budget, recent))
        self._in_order = [0 if n > budget else have for n, have in zip(self.lengths, self._in_order)]
        self.lengths = [min(n, budget) for n in self.lengths]
        self._give_back(range(len(self.lengths)))

    def release(self, b):
        """Sequence b is done: its pages are free, its place may be taken by another."""
        self.lengths[b] = self._in_order[b] = 0
        if self._positions is not None:
            self._positions[b] = 0
        self.seq_lens[b] = 0
        self.next_positions[b] = 0
        self._give_back([b])

    def _give_back(self, rows):
        page, changed = self.kv_pages.shape[2], []
        for b in rows:
            keep = -(-self.lengths[b] // page)
            if keep < len(self._pages[b]):
                self._free.extend(reversed(self._pages[b][keep:]))
                del self._pages[b][keep:]
                changed.append(b)
        if changed:
            self._write_table(changed)

    def _write_table(self, rows):
        width = self.block_table.shape[1]
        host = torch.tensor([self._pages[b] + [-1] * (width - len(self._pages[b])) for b in rows], dtype=torch.int32)
        if len(rows) == self.block_table.shape[0]:
            self.block_table.copy_(host)
        else:
            self.block_table[torch.tensor(rows, device=self.block_table.device)] = host.to(self.block_table.device)


class FineLlamaDecoderLayer:
    """forward(hidden_states [B, S, H], position_ids [B, S]) -> [B, S, H]; causal attention over the cache (if any)
    plus the new tokens. `weights`: dict of GPU tensors in nn.Linear layout: q, k, v, o, gate, up, down, and the norm
    weights ln1, ln2. `dtype` (float16 or bfloat16) is the type of the weights, activations and KV cache."""

    def __init__(self, weights, n_q_heads, n_kv_heads, rms_eps=1e-5, rope_base=10000.0, max_positions=8192,
                 dtype=torch.float16):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be float16 or bfloat16")
        self.dtype = dtype
        w = {k: v.detach().to(dtype).contiguous() for k, v in weights.items()}
        self.n_q, self.n_kv = int(n_q_heads), int(n_kv_heads)
        self.hidden = w["q"].shape[1]
        self.head_dim = w["q"].shape[0] // self.n_q
        if self.head_dim != 128:
            raise ValueError("head_dim must be 128, got %d" % self.head_dim)
        self.inter = w["gate"].shape[0]
        self.w_qkv = torch.cat((w["q"], w["k"], w["v"]), 0).contiguous()   # [(Hq + 2 Hkv) * D, H]
        self.w_o = w["o"]                                                  # [H, Hq * D]
        # gate and up rows interleaved in groups of 32, so the GEMM epilogue can apply silu(gate) * up to its accumulators
        self.gu_block = lib.GATE_UP_BLOCK if self.inter % lib.GATE_UP_BLOCK == 0 else 0
        self.w_gu = (lib.interleave_gate_up(w["gate"], w["up"]) if self.gu_block
                     else torch.cat((w["gate"], w["up"]), 0).contiguous())   # [2 F, H]
        self.w_d = w["down"]                                               # [H, F]
        self.ln1, self.ln2 = w["ln1"], w["ln2"]
        self.eps = float(rms_eps)
        self.cos, self.sin = rope_tables(max_positions, self.head_dim, rope_base, device=self.w_o.device)
        self.all_positions = torch.arange(max_positions, dtype=torch.int32, device=self.w_o.device)
        self.attn_ms = {"prefill": [], "decode": []}  # filled when time_attention=True (modeling_llama.py:762-775)

    @classmethod
    def from_hf(cls, hf_layer, config, max_positions=8192, device="cuda", dtype=torch.float16):
        """Wrap the weights of a transformers LlamaDecoderLayer."""
        a, m = hf_layer.self_attn, hf_layer.mlp
        w = dict(q=a.q_proj.weight, k=a.k_proj.weight, v=a.v_proj.weight, o=a.o_proj.weight, gate=m.gate_proj.weight,
                 up=m.up_proj.weight, down=m.down_proj.weight, ln1=hf_layer.input_layernorm.weight,
                 ln2=hf_layer.post_attention_layernorm.weight)
        w = {k: v.detach().to(device) for k, v in w.items()}
        base = getattr(config, "rope_theta", None) or (getattr(config, "rope_parameters", None) or {}).get("rope_theta", 10000.0)
        return cls(w, config.num_attention_heads, config.num_key_value_heads, config.rms_norm_eps, base, max_positions, dtype)

    def forward(self, hidden_states, position_ids=None, kv_cache=None, time_attention=False, new_lens=None):
        """With a FinePagedKVCache `new_lens` (a list) may say how many of each sequence's S rows are tokens, the first ones (none: all); the rows behind
        them must be finite and their results mean nothing. Its positions go on where each sequence's text is unless position_ids are given, behind
        which they go on from then."""
        B, S, H = hidden_states.shape
        if isinstance(kv_cache, FinePagedKVCache):
            return self._forward_paged(hidden_states, position_ids, kv_cache, time_attention, new_lens)
        if new_lens is not None:
            raise ValueError("new_lens goes with a FinePagedKVCache")
        past, kv, first = 0, (), 0
        if kv_cache is not None:
            past = kv_cache.length
            if past + S > kv_cache.max_len:
                raise ValueError("KV cache of %d tokens cannot take %d more after %d" % (kv_cache.max_len, S, past))
            # one tensor in the layout above, or any cache with `rows`, `k` and `v` as there
            kv = (kv_cache.kv,) if type(kv_cache) is FineKVCache else (kv_cache.rows(past, S), kv_cache.k, kv_cache.v)
        if position_ids is None:
            pos, first = self.all_positions, past   # a window of one table shared by every batch row, no kernel launched
            assert past + S <= pos.numel(), "max_positions is %d" % pos.numel()
        else:
            pos = position_ids.to(torch.int32).reshape(-1, S).contiguous()   # [1, S] (shared) or [B, S]
            assert pos.shape[0] in (1, B)
        out, ms = _C.layer_forward(hidden_states, self.w_qkv, self.w_o, self.w_gu, self.w_d, self.ln1, self.ln2, self.cos, self.sin, pos,
                                   first, kv, past, self.n_q, self.n_kv, self.eps, self.gu_block, time_attention, (), False)
        if kv_cache is not None:
            kv_cache.length = past + S
        if time_attention:
            self.attn_ms["decode" if (S == 1 and past > 0) else "prefill"].append(ms)
        return out

    def _forward_paged(self, hidden_states, position_ids, cache, time_attention, new_lens):
        B, S, _ = hidden_states.shape
        new = [S] * B if new_lens is None else [int(n) for n in new_lens]
        if len(new) != B or len(cache.lengths) != B or not all(0 <= n <= S for n in new):
            raise ValueError("%d sequences of up to %d new tokens, a cache of %d sequences and new_lens %r do not fit" % (B, S, len(cache.lengths), new_lens))
        if position_ids is None:
            if max(p + n for p, n in zip(cache.positions, new)) > self.cos.shape[0]:
                raise ValueError("max_positions is %d" % self.cos.shape[0])
            pos = cache.next_positions[:, None] + self.all_positions[:S]
        else:
            pos = position_ids.to(torch.int32).reshape(-1, S).contiguous()
            assert pos.shape[0] in (1, B)
        prompt = not any(cache.lengths)
        cache.extend(new)
        counts = None if all(n == S for n in new) else torch.tensor(new, dtype=torch.int32, device=hidden_states.device)
        paged = (cache.kv_pages, cache.table_in_use(S), cache.seq_lens, counts, cache.weights, cache.key_positions)
        try:
            out, ms = _C.layer_forward(hidden_states, self.w_qkv, self.w_o, self.w_gu, self.w_d, self.ln1, self.ln2, self.cos, self.sin, pos,
                                       0, (), 0, self.n_q, self.n_kv, self.eps, self.gu_block, time_attention, paged, prompt)
        except Exception:
            cache.take_back(new)
            raise
        if position_ids is not None:
            cache.went_to(pos, new)
        if time_attention:
            self.attn_ms["prefill" if prompt or S > 1 else "decode"].append(ms)
        return out

    __call__ = forward
