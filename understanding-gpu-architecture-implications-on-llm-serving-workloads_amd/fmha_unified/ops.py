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
           "fine_evict_paged"]

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
