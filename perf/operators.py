"""Performance cases of the paged key-value cache: its operators in plain torch operations and through the framework.

Four operators share one cache. It is a pool of pages [n_pages, 2 * Hkv, page, 128] (key heads in front of value heads), of which
each sequence owns those in its row of the block table: its key number j lies in page block_table[b][j // page], slot j % page.
`seq_lens` counts a sequence's keys, those of the call's tokens among them, which are its last ones. `new_lens` says how many of a
padded batch's rows are tokens (all of them without it). `weights` and `key_positions` [n_pages, Hkv, page] hold what eviction
goes by: the attention that a key has had so far, and the position of its token in the text.

    attend       softmax(scale q k^T + mask) v of one or a few new tokens of every sequence over its pages, with the log-sum-exp;
                 where `weights` is given, each key's probabilities, summed over its queries, are added to it
    write        rotary embedding of the queries and keys of a fused projection, keys and values filed into their pages
    key_weights  what the queries of a prompt (or its last rows) attended to, from their log-sum-exp: added to `weights`
    evict        every kv head of a sequence longer than the budget keeps the keys of the newest positions and, of the others, those
                 with the largest weights (ties: the lowest slot); kept keys that lie behind the budget move, in order, into the
                 slots of the dropped ones in front of it

    own                  False: plain forms in 32 bits; True: the calls that a user makes
    listed(), draw(rng)  the cases
    prepare(case, seed)  what a program holds before the call
    run(state)           one pass; returns everything it computes or changes
    exact(case, seed)    the same from the definitions, in 64 bits
    work(case)           bytes and flops that no implementation can do without

The working folder is the repository's root.
"""
import os
import sys

import torch

own = False

D = 128
SCALE = D ** -0.5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# ---- the cases -----------------------------------------------------------------------------------------------------


def _attend(B, Hq, Hkv, rows, longest, page, dtype="fp16", weights=False, ragged=False):
    return {"kind": "attend", "B": B, "Hq": Hq, "Hkv": Hkv, "rows": rows, "longest": longest, "page": page, "dtype": dtype,
            "weights": weights, "ragged": ragged}


def _write(B, Hq, Hkv, rows, past, page, dtype="fp16", ragged=False, keep_keys=False):
    return {"kind": "write", "B": B, "Hq": Hq, "Hkv": Hkv, "rows": rows, "past": past, "page": page, "dtype": dtype,
            "ragged": ragged, "keep_keys": keep_keys}


def _key_weights(B, Hq, Hkv, rows, past, last_rows, page, dtype="fp16", ragged=False):
    return {"kind": "key_weights", "B": B, "Hq": Hq, "Hkv": Hkv, "rows": rows, "past": past, "last_rows": last_rows,
            "page": page, "dtype": dtype, "ragged": ragged}


def _evict(B, Hkv, longest, budget, recent, page, dtype="fp16", ragged=False):
    return {"kind": "evict", "B": B, "Hkv": Hkv, "longest": longest, "budget": budget, "recent": recent, "page": page,
            "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # a generation step of one short sequence through a small layer: latency only
        dict(_attend(1, 8, 2, 1, 300, 16), name="attend_b1_300"),
        # a generation step of one sequence, odd number of cached keys
        dict(_attend(1, 32, 8, 1, 8191, 64), name="attend_b1_8191"),
        # four drafted tokens of each of four sequences are verified at once
        dict(_attend(4, 32, 8, 4, 2048, 32), name="attend_b4_rows4_2048"),
        # a step of 16 sequences of different lengths whose cache keeps account of what is attended to
        dict(_attend(16, 32, 8, 1, 4097, 32, weights=True, ragged=True), name="attend_weights_b16_4097"),
        # the largest step: a batch of a server, lengths from a few hundred keys to 8192, pages of 16 as they came free
        dict(_attend(64, 64, 8, 1, 8192, 16, "bf16", ragged=True), name="attend_b64_8192"),
        # the new tokens of a generation step are filed
        dict(_write(64, 32, 8, 1, 2048, 16, "bf16"), name="write_b64_step"),
        # prompts of different lengths, padded to the longest; their keys are read once more where they are
        dict(_write(4, 32, 8, 2048, 0, 16, ragged=True, keep_keys=True), name="write_prompts_4x2048"),
        # what the last 64 tokens of a prompt attended to
        dict(_key_weights(1, 32, 8, 64, 8127, 0, 16), name="key_weights_last64_8191"),
        # what all tokens of two prompts attended to
        dict(_key_weights(2, 32, 8, 4096, 0, 0, 32, "bf16"), name="key_weights_2x4096"),
        # 128 steps after the last eviction the caches of 16 sequences go back to 2048 keys
        dict(_evict(16, 8, 2176, 2048, 1024, 32, "bf16"), name="evict_b16_2176_to_2048"),
        # prompts of different lengths are cut to a quarter behind their prefill
        dict(_evict(4, 8, 8192, 2001, 64, 16, ragged=True), name="evict_prompts_8192_to_2001"),
    ]


def _log_uniform(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "write", "key_weights", "evict"))
    Hq, Hkv = rng.choice(((32, 8), (8, 2), (64, 8), (16, 4), (40, 8), (32, 32)))
    page, dtype, ragged = rng.choice((16, 32, 48, 64, 128)), rng.choice(("fp16", "bf16")), rng.random() < 0.6
    B = _log_uniform(rng, 1, 64)
    if kind == "attend":
        longest = _log_uniform(rng, 16, 32768)
        while B * longest * Hkv > 64 * 4096 * 8:
            B = max(1, B // 2) if B > 1 else B
            longest = longest if B > 1 else min(longest, 64 * 4096 * 8 // Hkv)
        rows = rng.choice((1, 1, 1, 2, 3, 4)) if Hq // Hkv * 4 <= 32 else 1
        return _attend(B, Hq, Hkv, min(rows, longest), longest, page, dtype, rng.random() < 0.4, ragged)
    if kind == "write":
        if rng.random() < 0.5:
            return _write(B, Hq, Hkv, rng.choice((1, 1, 2, 4)), _log_uniform(rng, 16, 4096), page, dtype, False, rng.random() < 0.3)
        rows = max(2, _log_uniform(rng, 16, 8192) // B)
        return _write(B, Hq, Hkv, rows, rng.choice((0, 0, 333)), page, dtype, ragged, rng.random() < 0.5)
    if kind == "key_weights":
        rows = max(2, _log_uniform(rng, 16, 4096) // B)
        past = rng.choice((0, 0, _log_uniform(rng, 16, 8192) // B))
        case = _key_weights(B, Hq, Hkv, rows, past, rng.choice((0, 0, min(rows, 32))), page, dtype, ragged)
        # none costs more than the largest listed
        return case if work(case)["flops"] <= 256 * 2 * 32 * 4096 * 4097 // 2 else draw(rng)
    budget = _log_uniform(rng, 64, 4096)
    longest = budget + rng.choice((1, 64, 128, budget, 3 * budget))
    while B * longest * Hkv > 16 * 8192 * 8 and B > 1:
        B //= 2
    return _evict(B, Hkv, longest, budget, budget // rng.choice((2, 4, 16)), page, dtype, ragged)


def _lengths(B, longest, ragged):
    """Keys (or tokens) of each sequence: `longest` of all, or the first that long and the others spread over [1/16, 1] of it."""
    spread = [1.0 if b == 0 or not ragged else 1 / 16 + 15 / 16 * ((b * 0.6180339887) % 1.0) for b in range(B)]
    return [max(1, int(longest * s)) for s in spread]


def _seq_and_new(case):
    """(seq_lens, new_lens, rows) of a case that brings tokens."""
    if case["kind"] == "attend":
        return _lengths(case["B"], case["longest"], case["ragged"]), [case["rows"]] * case["B"], case["rows"]
    new = _lengths(case["B"], case["rows"], case["ragged"])
    return [case["past"] + n for n in new], new, case["rows"]


# ---- inputs --------------------------------------------------------------------------------------------------------


def _cache(case, gen, seq_lens, fill=True):
    """A pool a little larger than its sequences need, whose pages are handed out in any order."""
    page, Hkv, B = case["page"], case["Hkv"], case["B"]
    per_seq = -(-max(seq_lens) // page)
    n_pages = B * per_seq + 3
    shape = (n_pages, 2 * Hkv, page, D)
    dtype = DTYPES[case["dtype"]]
    kv = torch.randn(shape, generator=gen, device="cuda", dtype=dtype) if fill else torch.zeros(shape, device="cuda", dtype=dtype)
    table = torch.randperm(n_pages, generator=gen, device="cuda")[:B * per_seq].reshape(B, per_seq).to(torch.int32)
    return {"kv_pages": kv, "block_table": table, "seq_lens": torch.tensor(seq_lens, dtype=torch.int32, device="cuda")}


def _account(state, gen, case):
    """What the keys have been attended to so far: most of them hardly, a few a lot."""
    n_pages = state["kv_pages"].shape[0]
    u = torch.rand((n_pages, case["Hkv"], case["page"]), generator=gen, device="cuda")
    return u.clamp_(min=1e-6).pow_(-0.7)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    B, Hkv, page, dtype = case["B"], case["Hkv"], case["page"], DTYPES[case["dtype"]]
    if case["kind"] == "evict":
        seq_lens = _lengths(B, case["longest"], case["ragged"])
        state = dict(_cache(case, gen, seq_lens), kind="evict", budget=case["budget"], recent=case["recent"])
        # positions: the text has gone on since the first tokens, keys lie where earlier evictions put them, each kv head's own
        slots = state["block_table"].shape[1] * page
        text = torch.rand((B, Hkv, slots + 1000), generator=gen, device="cuda").argsort(-1)[..., :slots].to(torch.int32)
        positions = torch.zeros((state["kv_pages"].shape[0], Hkv, page), dtype=torch.int32, device="cuda")
        positions[state["block_table"].long()] = text.reshape(B, Hkv, -1, page).transpose(1, 2)
        # both as they were before the pass, which is taken again from the same place
        state["account"] = torch.stack((_account(state, gen, case).view(torch.int32), positions))
        state["now"] = state["account"].clone()
        return state
    seq_lens, new_lens, rows = _seq_and_new(case)
    padded = case["kind"] != "attend" and case["ragged"]
    state = dict(_cache(case, gen, seq_lens, fill=case["kind"] != "write"), kind=case["kind"],
                 new_lens=torch.tensor(new_lens, dtype=torch.int32, device="cuda") if padded else None)
    n_pages = state["kv_pages"].shape[0]
    if case["kind"] == "write":
        heads = case["Hq"] + 2 * Hkv
        state["qkv"] = torch.randn((B, rows, heads, D), generator=gen, device="cuda", dtype=dtype)
        angle = torch.arange(case["past"] + rows + 700, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        # a sequence that was cut is further in its text than its cache is long
        ahead = torch.randint(0, 700, (B, 1), generator=gen, device="cuda")
        state["positions"] = (case["past"] + ahead + torch.arange(rows, device="cuda")).to(torch.int32)
        state["weights"] = _account(state, gen, case)
        state["key_positions"] = torch.zeros((n_pages, Hkv, page), dtype=torch.int32, device="cuda")
        return dict(state, q_heads=case["Hq"], keep_keys=case["keep_keys"])
    # queries a little longer than random ones: some keys get much of the attention
    state["q"] = torch.randn((B, rows, case["Hq"], D), generator=gen, device="cuda", dtype=dtype).mul_(1.5).transpose(1, 2)
    state["weights"] = None
    if case["kind"] == "key_weights" or case["weights"]:
        state["weights"] = _account(state, gen, case)
    if case["kind"] == "key_weights":
        state["last_rows"] = case["last_rows"]
        state["lse"] = _lse(state)
    return state


def _lse(state):
    """The log-sum-exp that the prompt's attention left, [B, Hq, rows]."""
    s, visible = _scores(state["q"], _keys(state, 0), state["seq_lens"], state["new_lens"])
    return s.masked_fill_(~visible[:, None, None], float("-inf")).logsumexp(-1).flatten(1, 2)


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _paged(x, table):
    """[n_pages, H, page, ...] -> [B, H, slots, ...]: the pages of every sequence one behind the other."""
    return x[table.long()].transpose(1, 2).flatten(2, 3)


def _keys(state, which):
    """Keys (0) or values (1) of every sequence in 32 bits, [B, Hkv, slots, 128]."""
    kv = state["kv_pages"]
    n = kv.shape[1] // 2
    return _paged(kv[:, which * n:(which + 1) * n], state["block_table"]).float()


def _scores(q, k, seq_lens, new_lens):
    """scale q k^T [B, Hkv, group, rows, slots], and which of them are visible [B, rows, slots]."""
    B, Hq, rows, _ = q.shape
    Hkv, slots = k.shape[1:3]
    s = torch.matmul(q.float().reshape(B, Hkv, -1, D), k.transpose(2, 3).contiguous()).mul_(SCALE).reshape(B, Hkv, Hq // Hkv, rows, slots)
    row, key = torch.arange(rows, device=q.device)[None, :, None], torch.arange(slots, device=q.device)
    new = torch.full_like(seq_lens, rows) if new_lens is None else new_lens
    return s, (key <= row + (seq_lens - new)[:, None, None]) & (row < new[:, None, None])


def _add_to_pages(pages, table, what, valid):
    """pages[table] += what [B, Hkv, slots] where valid [B, slots]."""
    page = pages.shape[2]
    where = table.long()
    old = pages[where]
    new = what.masked_fill(~valid[:, None], 0.0).unflatten(2, (-1, page)).transpose(1, 2)
    pages[where] = old + new


def _plain_attend(state):
    q, seq_lens = state["q"], state["seq_lens"]
    s, visible = _scores(q, _keys(state, 0), seq_lens, state["new_lens"])
    s.masked_fill_(~visible[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).flatten(1, 2).squeeze(-1)
    p.div_(total.clamp_(min=1e-38))
    if state["weights"] is not None:
        slots = torch.arange(p.shape[-1], device=q.device)
        _add_to_pages(state["weights"], state["block_table"], p.sum((2, 3)), slots < seq_lens[:, None])
    o = torch.matmul(p.flatten(2, 3), _keys(state, 1)).reshape(q.shape).to(q.dtype)
    return o, lse


def _plain_key_weights(state):
    q, seq_lens = state["q"], state["seq_lens"]
    s, visible = _scores(q, _keys(state, 0), seq_lens, state["new_lens"])
    rows, slots = s.shape[-2:]
    if state["last_rows"]:
        new = torch.full_like(seq_lens, rows) if state["new_lens"] is None else state["new_lens"]
        visible &= (torch.arange(rows, device=q.device) >= (new - state["last_rows"])[:, None])[..., None]
    lse = state["lse"].unflatten(1, s.shape[1:3])
    p = s.sub_(lse[..., None].clamp(min=-3e38)).exp_().masked_fill_(~visible[:, None, None], 0.0)
    _add_to_pages(state["weights"], state["block_table"], p.sum((2, 3)), torch.arange(slots, device=q.device) < seq_lens[:, None])


def _plain_write(state):
    qkv, kv, table = state["qkv"], state["kv_pages"], state["block_table"]
    B, rows, heads, _ = qkv.shape
    Hkv, page, n_q = kv.shape[1] // 2, kv.shape[2], state["q_heads"]
    c, s = state["cos"][state["positions"].long()][:, :, None], state["sin"][state["positions"].long()][:, :, None]
    x = qkv[:, :, :n_q + Hkv].float()
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    x = torch.cat((lo * c - hi * s, hi * c + lo * s), -1).to(qkv.dtype)
    new = state["new_lens"]
    new = torch.full_like(state["seq_lens"], rows) if new is None else new
    row = torch.arange(rows, device=qkv.device)
    token = row < new[:, None]                                  # [B, rows]
    kept = n_q + Hkv if state["keep_keys"] else n_q
    qkv[:, :, :kept] = torch.where(token[..., None, None], x[:, :, :kept], qkv[:, :, :kept])
    b, t = token.nonzero(as_tuple=True)
    slot = ((state["seq_lens"] - new)[:, None] + row)[b, t].long()
    where, at = table[b, slot // page].long(), slot % page
    kv[where, :Hkv, at] = x[b, t, n_q:]
    kv[where, Hkv:, at] = qkv[b, t, n_q + Hkv:]
    state["weights"][where, :, at] = 0.0
    state["key_positions"][where, :, at] = state["positions"][b, t][:, None]


def _plain_evict(state, weights, positions):
    kv, table, budget = state["kv_pages"], state["block_table"], state["budget"]
    Hkv, page = kv.shape[1] // 2, kv.shape[2]
    seq_lens = state["seq_lens"][:, None, None].long()
    w, pos = _paged(weights, table), _paged(positions, table).long()
    slot = torch.arange(w.shape[2], device=w.device)
    there = slot < seq_lens
    newest = pos.masked_fill(~there, -2 ** 40).amax(-1, keepdim=True)
    w = w.masked_fill(pos > newest - state["recent"], float("inf")).masked_fill(~there, float("-inf"))
    rank = torch.empty_like(pos).scatter_(2, w.sort(dim=-1, descending=True, stable=True).indices, slot.expand_as(pos))
    cut = seq_lens > budget
    keep = there & ((rank < budget) | ~cut)
    hole, moves = cut & ~keep & (slot < budget), cut & keep & (slot >= budget)
    # the n-th hole takes the n-th key that moves: nonzero() lists both in the order of (b, head, slot), equally many of each (b, head)
    b, h, to = hole.nonzero(as_tuple=True)
    _, _, at = moves.nonzero(as_tuple=True)
    to_page, to_slot = table[b, to // page].long(), to % page
    at_page, at_slot = table[b, at // page].long(), at % page
    kv[to_page, h, to_slot] = kv[at_page, h, at_slot]
    kv[to_page, h + Hkv, to_slot] = kv[at_page, h + Hkv, at_slot]
    weights[to_page, h, to_slot] = weights[at_page, h, at_slot]
    positions[to_page, h, to_slot] = positions[at_page, h, at_slot]
    return state["seq_lens"].clamp(max=budget)


# ---- a pass --------------------------------------------------------------------------------------------------------


def _ops():
    package = os.path.abspath("understanding-gpu-architecture-implications-on-llm-serving-workloads_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import fmha_unified
    return fmha_unified.ops


def run(state):
    cache = (state["kv_pages"], state["block_table"], state["seq_lens"])
    if state["kind"] == "attend":
        if own:
            o, lse = _ops().fine_fmha_paged_with_lse(state["q"], *cache, new_lens=state["new_lens"], weights=state["weights"])
        else:
            o, lse = _plain_attend(state)
        return {"o": o, "lse": lse, "weights": state["weights"]}
    if state["kind"] == "write":
        if own:
            _ops().fine_rope_paged(state["qkv"], *cache, state["cos"], state["sin"], state["positions"], state["q_heads"],
                                   new_lens=state["new_lens"], weights=state["weights"], key_positions=state["key_positions"],
                                   keep_keys=state["keep_keys"])
        else:
            _plain_write(state)
        return {name: state[name] for name in ("qkv", "kv_pages", "weights", "key_positions")}
    if state["kind"] == "key_weights":
        if own:
            _ops().fine_key_weights(state["q"], state["lse"], *cache, state["weights"], new_lens=state["new_lens"],
                                    last_rows=state["last_rows"])
        else:
            _plain_key_weights(state)
        return {"weights": state["weights"]}
    state["now"].copy_(state["account"])
    weights, positions = state["now"][0].view(torch.float32), state["now"][1]
    if own:
        lens = _ops().fine_evict_paged(*cache, weights, positions, state["budget"], state["recent"])
    else:
        lens = _plain_evict(state, weights, positions)
    return {"seq_lens": lens, "kv_pages": state["kv_pages"], "weights": weights, "key_positions": positions}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    table, lens, page, Hkv = st["block_table"].tolist(), st["seq_lens"].tolist(), case["page"], case["Hkv"]
    kv = st["kv_pages"]

    def places(b, n):
        """Pages and slots of the first n keys of sequence b."""
        j = torch.arange(n, device="cuda")
        return torch.tensor(table[b], device="cuda")[j // page], j % page

    if case["kind"] == "evict":
        weights, positions = st["account"][0].view(torch.float32).clone(), st["account"][1].clone()
        budget, left = case["budget"], list(lens)
        for b in range(case["B"]):
            if lens[b] <= budget:
                continue
            left[b] = budget
            pg, sl = places(b, lens[b])
            for h in range(Hkv):
                w, pos = weights[pg, h, sl].cpu().numpy(), positions[pg, h, sl].cpu().numpy().astype("int64")
                fresh = pos > pos.max() - case["recent"]
                # newest first, then by weight, then by slot
                order = sorted(range(lens[b]), key=lambda j: (not fresh[j], 0.0 if fresh[j] else -float(w[j]), j))
                kept = set(order[:budget])
                holes = [j for j in range(budget) if j not in kept]
                moved = [j for j in range(budget, lens[b]) if j in kept]
                d, s = torch.tensor(holes, device="cuda", dtype=torch.long), torch.tensor(moved, device="cuda", dtype=torch.long)
                for t, i in ((kv, h), (kv, h + Hkv), (weights, h), (positions, h)):
                    t[pg[d], i, sl[d]] = t[pg[s], i, sl[s]]
        return {"seq_lens": torch.tensor(left, dtype=torch.int32), "kv_pages": kv, "weights": weights, "key_positions": positions}
    _, new, rows = _seq_and_new(case)
    if case["kind"] == "write":
        qkv = st["qkv"].double()
        pages, weights, positions = kv.double(), st["weights"].double(), st["key_positions"].clone()
        n_q = case["Hq"]
        for b in range(case["B"]):
            pg, sl = places(b, lens[b])
            pg, sl, n = pg[-new[b]:], sl[-new[b]:], new[b]
            where = st["positions"][b, :n].long()
            turn = torch.complex(st["cos"][where].double(), st["sin"][where].double())[:, None]
            x = qkv[b, :n, :n_q + Hkv]
            y = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
            y = torch.cat((y.real, y.imag), -1)
            pages[pg, :Hkv, sl], pages[pg, Hkv:, sl] = y[:, n_q:], qkv[b, :n, n_q + Hkv:]
            qkv[b, :n, :n_q + Hkv * case["keep_keys"]] = y[:, :n_q + Hkv * case["keep_keys"]]
            weights[pg, :, sl], positions[pg, :, sl] = 0.0, st["positions"][b, :n, None]
        return {"qkv": qkv, "kv_pages": pages, "weights": weights, "key_positions": positions}
    group = case["Hq"] // Hkv
    weights = None if st["weights"] is None else st["weights"].double()
    o, lse = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64), torch.zeros(st["q"].shape[:3], device="cuda", dtype=torch.float64)
    for b in range(case["B"]):
        pg, sl = places(b, lens[b])
        for h in range(Hkv):
            k, v = kv[pg, h, sl].double(), kv[pg, Hkv + h, sl].double()
            for i in range(h * group, (h + 1) * group):
                s = st["q"][b, i, :new[b]].double() @ k.T / D ** 0.5
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(lens[b] - new[b] + 1), float("-inf"))
                if case["kind"] == "attend":
                    lse[b, i] = s.logsumexp(-1)
                    p = s.softmax(-1).nan_to_num(0.0)   # a row that sees no key gives zeros
                    o[b, i] = p @ v
                else:
                    p = (s - st["lse"][b, i, :new[b], None].double()).exp()[-case["last_rows"]:]
                if weights is not None:
                    weights[pg, h, sl] += p.sum(0)
    return {"o": o, "lse": lse, "weights": weights} if case["kind"] == "attend" else {"weights": weights}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def _visible(new, length, last_rows=0):
    """Pairs of a query and a key that it sees, of one sequence."""
    first = max(0, new - last_rows) if last_rows else 0
    return sum(max(0, i + length - new + 1) for i in range(first, new))


def work(case):
    B, Hkv = case["B"], case["Hkv"]
    if case["kind"] == "evict":
        cut = [n for n in _lengths(B, case["longest"], case["ragged"]) if n > case["budget"]]
        # weights and positions of all keys; of the keys that move (how many is for the data to say: the expected number of a
        # random choice) the key, the value, the weight and the position are read and written
        moved = sum(case["budget"] * (n - case["budget"]) / n for n in cut)
        return {"bytes": int(Hkv * (8 * sum(cut) + 2 * moved * (4 * D + 8))), "flops": 0}
    lens, new, rows = _seq_and_new(case)
    if case["kind"] == "write":
        tokens = sum(new)
        heads = case["Hq"] + 2 * Hkv
        written = heads + (Hkv if case["keep_keys"] else 0)
        return {"bytes": tokens * (2 * D * (heads + written) + 8 * D // 2 + 4 + 8 * Hkv), "flops": 6 * tokens * (case["Hq"] + Hkv) * D // 2}
    if case["kind"] == "key_weights":
        last = case["last_rows"]
        read = sum(min(n, last) if last else n for n in new)
        return {"bytes": 2 * D * (Hkv * sum(lens) + case["Hq"] * read) + 4 * case["Hq"] * read + 8 * Hkv * sum(lens),
                "flops": 2 * D * case["Hq"] * sum(_visible(n, t, last) for n, t in zip(new, lens))}
    return {"bytes": 4 * D * Hkv * sum(lens) + 4 * D * case["Hq"] * rows * B + 4 * case["Hq"] * rows * B + (8 * Hkv * sum(lens) if case["weights"] else 0),
            "flops": 4 * D * case["Hq"] * sum(_visible(n, t) for n, t in zip(new, lens))}
