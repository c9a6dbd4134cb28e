"""Python entry point of the attention operators; mirrors kernels/fmha/pkg/fmha_unified/ops.py:8-29.

The reference pads q, k and v to a multiple of 64 rows with ``F.pad`` (a full copy of each tensor, ops.py:19-25),
passes the un-padded key count as ``decode_length`` (ops.py:18,27) and slices the output back (ops.py:29). The
MI355X kernel masks ragged tails itself, so nothing is padded, copied or sliced here; the result is the same.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _C

__all__ = ["fine_fmha", "fine_fmha_with_lse", "fine_fmha_paged", "fine_fmha_paged_with_lse", "fine_rope_paged", "fine_key_weights",
           "fine_evict_paged", "fine_fmha_tree", "fine_fmha_tree_with_lse", "fine_keep_path", "fine_plan_packed", "fine_rope_packed", "fine_fmha_packed",
           "fine_fmha_packed_with_lse"]

# the operators of all indices, looked up by name once
_KERNELS = {i: getattr(torch.ops.fmha_unified, f"finefmha_{i}").default for i in range(8)}


def fine_fmha(q: Tensor, k: Tensor, v: Tensor, causal: bool, is_decode, kernel_index: int) -> Tensor:
    """softmax(q k^T / sqrt(d) + mask) v for q [B,Hq,Sq,128], k, v [B,Hkv,Sk,128] (fp16, GPU).

    ``causal`` masks key j for query i when j > i + (Sk - Sq); ``is_decode`` (requires ``causal=False``) is the
    single-query generation step. GQA: query head h uses kv head h // (Hq // Hkv).

    Difference from the reference for ``Sq != Sk``: its kernels mask key j when j > i (top-left alignment,
    semi/fmha_2_amd.cpp:187-190); here the mask is aligned to the bottom-right corner (the KV-cache convention). The two
    are the same mask when ``Sq == Sk``, the only causal case the reference's tests and drivers use. A query row with no
    visible key (``Sq > Sk`` only) gives zeros. The result is a new contiguous [B, Hq, Sq, 128] tensor.
    """
    kernel = _KERNELS.get(kernel_index) if type(kernel_index) is int else None
    if kernel is None:
        kernel = getattr(torch.ops.fmha_unified, f"finefmha_{int(kernel_index)}").default
    decode_length = k.size(2)
    return kernel(q, k, v, bool(causal), bool(is_decode), decode_length)


def fine_fmha_with_lse(q: Tensor, k: Tensor, v: Tensor, causal: bool, is_decode=False) -> Tuple[Tensor, Tensor]:
    """As :func:`fine_fmha`, also returning the fp32 log-sum-exp [B,Hq,Sq] of the scaled, masked scores."""
    return torch.ops.fmha_unified.finefmha_fwd_lse.default(q, k, v, bool(causal), bool(is_decode), k.size(2))


# ---- a key-value cache in pages ------------------------------------------------------------------------------------
#
# kv_pages     [n_pages, 2 * Hkv, page_size, 128] fp16 or bf16: the pool of pages, key heads in front of value heads (any strides with a
#              contiguous last dimension); page_size a multiple of 16
# block_table  [B, max_pages] int32: key j of sequence b lies in page block_table[b][j // page_size], slot j % page_size; entries
#              outside the pool hold no keys
# seq_lens     [B] int32: keys of each sequence, those of this call's tokens among them, which are its last ones
# new_lens     [B] int32 or None: how many of the S rows of a padded batch are tokens, the first ones (None: all S)
# weights, key_positions   [n_pages, Hkv, page_size] fp32 and int32: the attention each key has had, the position of its token
#
# Everything is read on the device: no call waits for it, and a captured call serves the lengths and tables that its tensors hold
# when the graph is replayed. No page may belong to two sequences of a call that writes it, to its weights among others. Hq / Hkv * S is below
# 2^24 (2^16 where S is more than max_pages * page_size); the other limits are those of include/mi355_serving.h. The reference keeps one
# growing tensor a layer instead (benchmarks/flashattn-cuda/modeling_llama.py:664-668).

# The functions below call the extension module's own (which ask the dispatcher where a mode, a transform, a tracer or a gradient that is needed would not see
# them otherwise); `torch.ops.fmha_unified.{finefmha_paged, finefmha_paged_lse, rope_paged, key_weights, evict_paged}` are the same through torch's
# dispatcher. Inference only: there is no backward.

def fine_fmha_paged(q: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, new_lens: Optional[Tensor] = None,
                    weights: Optional[Tensor] = None) -> Tensor:
    """softmax(q k^T / sqrt(d) + mask) v for the S rows of every sequence, q [B, Hq, S, 128], over its pages: the new token of a
    generation step, a few drafted ones, a chunk of a prompt. Row i of `new` tokens is key seq_lens[b] - new + i and sees the keys up to that
    one; a row that sees none, or is no token, gives zeros. With `weights`, each key's probabilities, summed over the query heads of its
    kv head and the rows, are added to it. The result is a new contiguous [B, Hq, S, 128] tensor."""
    return _C.finefmha_paged(q, kv_pages, block_table, seq_lens, new_lens, weights)


def fine_fmha_paged_with_lse(q: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, new_lens: Optional[Tensor] = None,
                             weights: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """As :func:`fine_fmha_paged`, also returning the fp32 log-sum-exp [B, Hq, S] of the scaled, masked scores."""
    return _C.finefmha_paged_lse(q, kv_pages, block_table, seq_lens, new_lens, weights)


def fine_rope_paged(qkv: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, cos: Tensor, sin: Tensor, positions: Tensor,
                    q_heads: int, new_lens: Optional[Tensor] = None, weights: Optional[Tensor] = None,
                    key_positions: Optional[Tensor] = None, keep_keys: bool = False) -> None:
    """Rotary embedding of a fused projection qkv [B, S, q_heads + 2 * Hkv, 128] with its keys and values filed into their pages: the query
    heads are rotated in place, token t becomes key seq_lens[b] - new + t. cos, sin: [n_positions, 64] fp32; positions: int32, [B, S] or [S]
    (shared by all sequences). Where they are given, the new keys' `weights` become zero and their `key_positions` the tokens'
    positions. keep_keys: the rotated keys are stored in qkv as well."""
    _C.rope_paged(qkv, kv_pages, block_table, seq_lens, cos, sin, positions, q_heads, new_lens, weights, key_positions, keep_keys)


def fine_key_weights(q: Tensor, lse: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, weights: Tensor,
                     new_lens: Optional[Tensor] = None, last_rows: int = 0) -> None:
    """What a prompt's rows attended to is added to `weights`: for every key the sum of exp(q k / sqrt(d) - lse) over the query heads of its
    kv head and the rows that see it. q [B, Hq, S, 128] and lse [B, Hq, S] are those of the attention over the same keys. last_rows > 0:
    only the last that many tokens of each sequence count."""
    _C.key_weights(q, lse, kv_pages, block_table, seq_lens, weights, new_lens, last_rows)


def fine_evict_paged(kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, weights: Tensor, key_positions: Tensor, budget: int,
                     recent: int) -> Tensor:
    """Cuts sequences longer than `budget` to it, every kv head on its own: kept are the keys whose position is within `recent` of the
    largest, then those of the largest weights (NaN lowest), of equals the lowest slots. Kept keys that lie behind the budget move, in order,
    into the slots of dropped ones in front of it, with their values, weights and positions. Returns the new lengths, min(seq_lens,
    budget); seq_lens itself is left as it is, and so are the slots from `budget` on. Slots of pages outside the pool hold no key and take
    none: where there are some in front of the budget, so many keys fewer are kept."""
    return _C.evict_paged(kv_pages, block_table, seq_lens, weights, key_positions, budget, recent)


# ---- a tree of drafted tokens ----------------------------------------------------------------------------------------
#
# The S rows of a call (S <= 256) are drafted tokens, the last keys of their sequence: row i continues row parents[b][i] (0 <= parent < i; anything else makes it a
# root). File them with fine_rope_paged, at the positions of their depths; then attend with fine_fmha_tree, and close ranks with fine_keep_path once
# it is known which were accepted. No account (`weights`) is kept of drafted tokens.

def fine_fmha_tree(q: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, parents: Tensor, new_lens: Optional[Tensor] = None) -> Tensor:
    """:func:`fine_fmha_paged` for a tree of drafted tokens, q [B, Hq, S, 128]: a row sees the keys in front of the draft, itself and the rows on its path to a
    root. parents: int32, [B, S] or [S] (shared by all sequences). The result is a new contiguous [B, Hq, S, 128] tensor."""
    return _C.fmha_tree(q, kv_pages, block_table, seq_lens, parents, new_lens)


def fine_fmha_tree_with_lse(q: Tensor, kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, parents: Tensor,
                            new_lens: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """As :func:`fine_fmha_tree`, also returning the fp32 log-sum-exp [B, Hq, S] of the scaled, masked scores."""
    return _C.fmha_tree_lse(q, kv_pages, block_table, seq_lens, parents, new_lens)


def fine_keep_path(kv_pages: Tensor, block_table: Tensor, seq_lens: Tensor, new_lens: Tensor, path: Tensor, weights: Optional[Tensor] = None,
                   key_positions: Optional[Tensor] = None) -> Tensor:
    """Of the last new_lens[b] keys of each sequence, drafted tokens, those of `path` [B, length] (int32, ascending, ending in front of the first entry that does not
    ascend or is no drafted token, so -1 behind the last) move, with their values, weights and positions, to the places behind the keys in front of the
    draft. Returns the new lengths; seq_lens itself is left as it is, and so are the keys behind them."""
    return _C.keep_path(kv_pages, block_table, seq_lens, new_lens, path, weights, key_positions)


# ---- packed batches --------------------------------------------------------------------------------------------------
#
# The tokens of sequences of different lengths lie one behind the other, [rows, ...] without padding: sequence b has rows offsets[b] .. offsets[b + 1] - 1 (int32,
# on the device, ascending from 0). Rows behind the last sequence are no tokens. As above nothing waits for the device, and a captured call serves what its
# tensors hold when the graph is replayed. The exact rules and the limits are in include/mi355_serving.h.

def fine_plan_packed(block_table: Tensor, seq_lens: Tensor, new_lens: Tensor, free_pages: Tensor, free_span: Tensor, page_size: int, rows: int,
                     next_positions: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """Block tables and slot maps from the lengths of the requests: new_lens[b] tokens come to sequence b, which has seq_lens[b] keys. Pages that its row of
    block_table lacks are taken from the ring `free_pages` [n_pages], which holds free_span[1] pages from place free_span[0] on; pages behind its end go back
    there. block_table, seq_lens, free_pages, free_span and next_positions (the position of each sequence's next token; without them a token's position is the number of its
    key) are brought up to date. All tensors are int32.

    Returns offsets [B + 1] of a packed batch of `rows` rows, the position and the slot (page * page_size + row of the page) of each row's token, -1 where there is none, and
    `taken` [B]: new_lens, or 0 where the sequence has no room in its row of the table or in the batch, or the ring not the pages that it and those in front of it
    lack; such a sequence stays as it is. seq_lens[b] = 0 with new_lens[b] = 0 releases a sequence's pages.

    A new pool: block_table full of -1, seq_lens 0, free_pages = arange(n_pages), free_span = [0, n_pages]."""
    return _C.plan_packed(block_table, seq_lens, new_lens, free_pages, free_span, page_size, rows, next_positions)


def fine_rope_packed(qkv: Tensor, kv_pages: Tensor, slots: Tensor, cos: Tensor, sin: Tensor, positions: Tensor, q_heads: int, weights: Optional[Tensor] = None,
                     key_positions: Optional[Tensor] = None, keep_keys: bool = True) -> None:
    """:func:`fine_rope_paged` for a packed batch, qkv [rows, q_heads + 2 * Hkv, 128]: row t is the token at positions[t] (negative: no token, the row stays as it is),
    whose key and value go to slot slots[t] of the pool (outside it: they are not filed). keep_keys: the rotated keys are stored in qkv as well, where
    :func:`fine_fmha_packed` reads them."""
    _C.rope_packed(qkv, kv_pages, slots, cos, sin, positions, q_heads, weights, key_positions, keep_keys)


def fine_fmha_packed(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, causal: bool = True) -> Tensor:
    """softmax(q k^T / sqrt(d) + mask) v of each sequence's rows over its own rows, q [rows, Hq, 128], k, v [rows, Hkv, 128] (slices of one fused projection will do);
    causal: row i sees the rows 0 .. i of its sequence. Rows that no sequence has give zeros. The result is a new contiguous [rows, Hq, 128] tensor."""
    return _C.fmha_packed(q, k, v, offsets, causal)


def fine_fmha_packed_with_lse(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, causal: bool = True) -> Tuple[Tensor, Tensor]:
    """As :func:`fine_fmha_packed`, also returning the fp32 log-sum-exp [Hq, rows] of the scaled, masked scores (-inf in rows that no sequence has)."""
    return _C.fmha_packed_lse(q, k, v, offsets, causal)
