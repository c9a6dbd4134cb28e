"""Performance cases of packed batches and drafted trees: their operators in plain torch operations and through the framework.

A packed batch holds the tokens of its sequences one behind the other, [rows, ...] without padding: those of sequence b are rows
offsets[b] .. offsets[b + 1] - 1. Their keys and values go to a pool of pages [n_pages, 2 * Hkv, page, 128] (key heads in front of
value heads); key j of sequence b lies in page block_table[b][j // page], slot j % page. Pages that no sequence has are listed in a
ring, free_pages, of which free_span says the first place and the count.

    plan    the lengths of the requests become the block table (pages taken from the ring where new tokens need them, given back
            behind the sequences' ends), the offsets, and position and slot (page * page size + row of the page) of every token
    rope    rotary embedding of the queries and keys of a packed projection, keys and values filed into their slots
    packed  attention of whole prompts, causal or not: softmax(scale q k^T + mask) v and the log-sum-exp
    tree    attention of a tree of drafted tokens, which are a sequence's last keys, over its pages: a token sees the keys in front
            of the tree, itself and what it descends from (parents[b][i] < i; a root's is negative)
    keep    the accepted path of a tree: its keys and values close ranks behind the keys in front of the tree

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


def _packed(B, Hq, Hkv, longest, dtype="fp16", ragged=True, causal=True, spare=0):
    return {"kind": "packed", "B": B, "Hq": Hq, "Hkv": Hkv, "longest": longest, "dtype": dtype, "ragged": ragged, "causal": causal, "spare": spare}


def _plan(B, longest, prompts, page, columns, spare=0):
    return {"kind": "plan", "B": B, "longest": longest, "prompts": prompts, "page": page, "columns": columns, "spare": spare}


def _rope(B, Hq, Hkv, longest, page, dtype="fp16", ragged=True, spare=0):
    return {"kind": "rope", "B": B, "Hq": Hq, "Hkv": Hkv, "longest": longest, "page": page, "dtype": dtype, "ragged": ragged, "spare": spare}


def _tree(B, Hq, Hkv, nodes, longest, page, dtype="fp16", ragged=False, some=False):
    return {"kind": "tree", "B": B, "Hq": Hq, "Hkv": Hkv, "nodes": nodes, "longest": longest, "page": page, "dtype": dtype, "ragged": ragged, "some": some}


def _keep(B, Hkv, nodes, longest, page, dtype="fp16", account=False):
    return {"kind": "keep", "B": B, "Hkv": Hkv, "nodes": nodes, "longest": longest, "page": page, "dtype": dtype, "account": account}


def listed():
    return [
        # three short prompts through a small layer: latency only
        dict(_packed(3, 8, 2, 77), name="packed_b3_77"),
        # the prompts of one step of a server, lengths from 64 to 1000 tokens, the projection padded at its end
        dict(_packed(16, 32, 8, 1000, "bf16", spare=45), name="packed_b16_1000"),
        # the largest: a long prompt and shorter ones
        dict(_packed(4, 32, 8, 8192), name="packed_b4_8192"),
        # the next token of 64 running requests: every sixteenth needs a page
        dict(_plan(64, 8000, 0, 16, 512), name="plan_step_b64"),
        # 256 requests, a quarter of them with new prompts, some done, whose pages come back
        dict(_plan(256, 1500, 64, 32, 1024, spare=77), name="plan_prompts_b256"),
        # the tokens of a generation step are rotated and filed
        dict(_rope(64, 32, 8, 1, 16, "bf16", ragged=False), name="rope_step_b64"),
        # the prompts of a step, about 8000 tokens
        dict(_rope(8, 32, 8, 2048, 16, spare=100), name="rope_prompts_8x2048"),
        # 26 drafted tokens of one short sequence through a small layer: latency
        dict(_tree(1, 8, 2, 26, 300, 16), name="tree_b1_26_300"),
        # 64 drafted tokens of a long sequence, odd number of keys
        dict(_tree(1, 32, 8, 64, 8191, 64), name="tree_b1_64_8191"),
        # drafts of different sizes of 32 sequences of different lengths
        dict(_tree(32, 32, 8, 32, 4097, 32, "bf16", ragged=True, some=True), name="tree_b32_32_4097"),
        # accepted paths through small drafts
        dict(_keep(4, 8, 26, 700, 16), name="keep_b4_26"),
        # the same of a server's batch, larger drafts, with the account that eviction goes by
        dict(_keep(64, 8, 64, 2048, 32, "bf16", account=True), name="keep_b64_64"),
    ]


def _log_uniform(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("packed", "packed", "tree", "tree", "plan", "rope", "keep"))
    Hq, Hkv = rng.choice(((32, 8), (8, 2), (64, 8), (16, 4), (40, 8), (32, 32)))
    page, dtype = rng.choice((16, 32, 48, 64, 128)), rng.choice(("fp16", "bf16"))
    spare = rng.choice((0, 0, 1, 130))
    B = _log_uniform(rng, 1, 64)
    if kind == "packed":
        longest = _log_uniform(rng, 1, 6000)
        while B * Hq * longest * longest > 2 * 32 * 6000 * 6000:
            B, longest = max(1, B // 2), longest if B > 1 else longest // 2
        return _packed(B, Hq, Hkv, longest, dtype, rng.random() < 0.8, rng.random() < 0.8, spare)
    if kind == "plan":
        B = _log_uniform(rng, 1, 1000)
        longest = _log_uniform(rng, 8, 3000)
        prompts = rng.choice((0, B, rng.randint(0, B)))
        while prompts * longest > 64 * 1500:
            prompts //= 2
        return _plan(B, longest, prompts, page, 2 * longest // page + rng.randint(3, 300), spare)
    if kind == "rope":
        longest = rng.choice((1, max(1, _log_uniform(rng, 16, 8192) // B)))
        return _rope(B, Hq, Hkv, longest, page, dtype, rng.random() < 0.7, spare)
    nodes = _log_uniform(rng, 2, 128)
    longest = _log_uniform(rng, 16, 16384) + nodes
    if kind == "keep":
        while B * longest * Hkv > 64 * 2048 * 8 and B > 1:
            B //= 2
        return _keep(B, Hkv, nodes, min(longest, 4096), page, dtype, rng.random() < 0.5)
    while B * longest * Hkv > 32 * 4096 * 8 or B * nodes * longest * Hq > 32 * 32 * 4096 * 32:
        if B > 1:
            B //= 2
        else:
            longest = longest // 2 + nodes
            nodes = max(2, nodes // 2)
    return _tree(B, Hq, Hkv, nodes, longest, page, dtype, rng.random() < 0.6, rng.random() < 0.4)


def _lengths(B, longest, ragged):
    """Tokens of each sequence: `longest` of all, or the first that long and the others spread over [1/16, 1] of it."""
    spread = [1.0 if b == 0 or not ragged else 1 / 16 + 15 / 16 * ((b * 0.6180339887) % 1.0) for b in range(B)]
    return [max(1, int(longest * s)) for s in spread]


def _requests(case):
    """(keys so far, new tokens) of each request of a plan: prompts at the front, running ones, every eleventh done."""
    B, longest = case["B"], case["longest"]
    lens = _lengths(B, longest, True)
    prompt = [b < case["prompts"] for b in range(B)]
    done = [not p and b % 11 == 7 for b, p in enumerate(prompt)]
    past = [0 if p or d else n for n, p, d in zip(lens, prompt, done)]
    return past, [n if p else 0 if d else 1 for n, p, d in zip(lens, prompt, done)]


def _drafts(case):
    """(keys, drafted tokens among them) of each sequence of a tree."""
    B, nodes = case["B"], case["nodes"]
    lens = [max(n, nodes) for n in _lengths(B, case["longest"], case.get("ragged", True))]
    return lens, _lengths(B, nodes, bool(case.get("some")))


# ---- inputs --------------------------------------------------------------------------------------------------------


def _pool(case, gen, per_seq):
    """Pages in any order: a table of per_seq columns for every sequence, and a pool a little larger."""
    B, n_pages = case["B"], case["B"] * per_seq + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    return order[:B * per_seq].reshape(B, per_seq), n_pages


def _kv_pages(case, gen, n_pages, fill=True):
    shape, dtype = (n_pages, 2 * case["Hkv"], case["page"], D), DTYPES[case["dtype"]]
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype) if fill else torch.zeros(shape, device="cuda", dtype=dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    return _ints([sum(lens[:b]) for b in range(len(lens) + 1)])


def _prepare_plan(case, gen):
    B, page, columns = case["B"], case["page"], case["columns"]
    past, new = _requests(case)
    # pages of what a sequence has had: a running one's keys, a few more where drafted tokens were not accepted, a done one's
    had = _lengths(B, case["longest"], True)
    held = [0 if b < case["prompts"] else -(-(n + 16 * (b % 5 == 2)) // page) for b, n in enumerate(had)]
    wanted = sum(max(0, -(-(p + n) // page) - h) for p, n, h in zip(past, new, held))
    n_pages = sum(held) + wanted + 10
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    column, first = torch.arange(columns, device="cuda"), torch.tensor([sum(held[:b]) for b in range(B)], device="cuda")
    there = column < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(there, order[(first[:, None] + column).clamp(max=n_pages - 1)], torch.full_like(column, -1, dtype=torch.int32))
    count, at = n_pages - sum(held), int(torch.randint(0, n_pages, (1,), generator=gen, device="cuda"))
    ring = torch.roll(torch.cat((order[sum(held):], torch.full((sum(held),), -1, dtype=torch.int32, device="cuda"))), at)
    # all that a plan changes, as it was before the pass, which is taken again from the same place
    texts = torch.randint(0, 700, (B,), generator=gen, device="cuda").to(torch.int32) + _ints(past)   # (a cut sequence is further in its text)
    saved = torch.cat((table.reshape(-1), _ints(past), ring, _ints([at, count]), texts))
    now = saved.clone()
    sizes = (B * columns, B, n_pages, 2, B)
    views = dict(zip(("block_table", "seq_lens", "free_pages", "free_span", "next_positions"), now.split(sizes)))
    views["block_table"] = views["block_table"].view(B, columns)
    return dict(views, kind="plan", saved=saved, now=now, new_lens=_ints(new), page=page, rows=sum(new) + case["spare"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, B = case["kind"], case["B"]
    if kind == "plan":
        return _prepare_plan(case, gen)
    Hkv, dtype = case["Hkv"], DTYPES[case["dtype"]]
    if kind in ("packed", "rope"):
        lens = _lengths(B, case["longest"], case["ragged"])
        rows, heads = sum(lens) + case["spare"], case["Hq"] + 2 * Hkv
        qkv = torch.randn((rows, heads, D), generator=gen, device="cuda", dtype=dtype)
        if kind == "packed":
            # queries a little longer than random ones: some keys get much of the attention
            qkv[:, :case["Hq"]].mul_(1.5)
            q, k, v = qkv.split((case["Hq"], Hkv, Hkv), 1)
            return {"kind": kind, "q": q, "k": k, "v": v, "offsets": _offsets(lens), "longest": max(lens), "causal": case["causal"]}
        page = case["page"]
        past = 37   # keys in front of the new tokens
        table, n_pages = _pool(case, gen, -(-(past + max(lens)) // page))
        sequence = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(lens, device="cuda"))
        key = past + torch.arange(sum(lens), device="cuda") - _offsets(lens).long()[sequence]
        slots = table[sequence, key // page] * page + key % page
        ahead = torch.randint(0, 700, (B,), generator=gen, device="cuda")   # (a cut sequence is further in its text)
        none = torch.full((case["spare"],), -1, device="cuda")
        angle = torch.arange(past + max(lens) + 700, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
        shape = (n_pages, Hkv, page)
        return {"kind": kind, "qkv": qkv, "kv_pages": _kv_pages(case, gen, n_pages, fill=False), "slots": torch.cat((slots, none)).to(torch.int32),
                "positions": torch.cat((key + ahead[sequence], none)).to(torch.int32), "cos": angle.cos().float(), "sin": angle.sin().float(),
                "q_heads": case["Hq"], "weights": torch.rand(shape, generator=gen, device="cuda"),
                "key_positions": torch.zeros(shape, dtype=torch.int32, device="cuda")}
    lens, new = _drafts(case)
    table, n_pages = _pool(case, gen, -(-max(lens) // case["page"]))
    nodes = case["nodes"]
    state = {"kind": kind, "kv_pages": _kv_pages(case, gen, n_pages), "block_table": table, "seq_lens": _ints(lens)}
    if kind == "tree":
        # a token continues one of the eight drafted before it (the first one, and now and then another, is a root)
        node = torch.arange(nodes, device="cuda")
        back = torch.randint(1, 9, (B, nodes), generator=gen, device="cuda")
        state["parents"] = (node - back).clamp(min=-1).to(torch.int32)
        state["new_lens"] = _ints(new) if case["some"] else None
        state["q"] = torch.randn((B, nodes, case["Hq"], D), generator=gen, device="cuda", dtype=dtype).mul_(1.5).transpose(1, 2)
        return state
    # from each drafted token accepted one goes on a few further: ascending numbers, -1 behind the last
    length = -(-nodes // 4)
    steps = torch.randint(1, 6, (B, length), generator=gen, device="cuda")
    path = steps.cumsum(1) - 1
    accepted = torch.randint(1, length + 1, (B, 1), generator=gen, device="cuda")
    state["path"] = path.masked_fill((path >= nodes) | (torch.arange(length, device="cuda") >= accepted), -1).to(torch.int32)
    state["new_lens"] = _ints(new)
    shape = (n_pages, Hkv, case["page"])
    state["weights"] = torch.rand(shape, generator=gen, device="cuda") if case["account"] else None
    state["key_positions"] = torch.randint(0, 1 << 20, shape, generator=gen, device="cuda").to(torch.int32) if case["account"] else None
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _attention(q, k, v, visible):
    """q [B, Hq, N, 128], k, v [B, Hkv, S, 128] in 32 bits, visible [B, N, S] -> o in 32 bits, lse; a row that sees nothing gives zeros."""
    B, Hq, N, _ = q.shape
    Hkv, S = k.shape[1:3]
    s = torch.matmul(q.reshape(B, Hkv, -1, D), k.transpose(2, 3).contiguous()).mul_(SCALE).reshape(B, Hkv, Hq // Hkv, N, S)
    s.masked_fill_(~visible[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).flatten(1, 2).squeeze(-1)
    p.div_(total.clamp_(min=1e-38))
    return torch.matmul(p.flatten(2, 3), v).reshape(q.shape), lse


def _plain_packed(state):
    q, offsets, longest = state["q"], state["offsets"].long(), state["longest"]
    begin, lens = offsets[:-1], offsets[1:] - offsets[:-1]
    t = torch.arange(longest, device=q.device)
    token = t < lens[:, None]                                       # [B, longest]
    at = (begin[:, None] + t).clamp(max=q.shape[0] - 1)
    qp, kp, vp = (state[x][at].float().transpose(1, 2).contiguous() for x in ("q", "k", "v"))
    visible = token[:, None, :] & token[:, :, None]
    if state["causal"]:
        visible &= t[None, :] <= t[:, None]
    op, lsep = _attention(qp, kp, vp, visible)
    o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.full((q.shape[1], q.shape[0]), float("-inf"), device=q.device)
    rows = at[token]
    o[rows] = op.transpose(1, 2)[token].to(q.dtype)
    lse[:, rows] = lsep.transpose(1, 2)[token].T
    return o, lse


def _plain_plan(state):
    table, ring, span, page, rows = state["block_table"], state["free_pages"], state["free_span"], state["page"], state["rows"]
    B, columns = table.shape
    n_pages = ring.numel()
    past, new = state["seq_lens"].long().clamp(0, columns * page), state["new_lens"].long().clamp(min=0)
    end = new.cumsum(0)
    held, column = (table >= 0) & (table < n_pages), torch.arange(columns, device=table.device)
    fits = (past + new <= columns * page) & (end <= rows)
    wanted = ~held & (column >= (past // page)[:, None]) & (column < ((past + new + page - 1) // page)[:, None]) & (fits & (new > 0))[:, None]
    lacks = wanted.sum(1)
    admitted = fits & ((lacks == 0) | (lacks.cumsum(0) <= span[1]))
    taken = new * admitted
    wanted &= admitted[:, None]
    first, count = span[0].long(), span[1].long()
    number = wanted.flatten().cumsum(0).view(B, columns)
    table.copy_(torch.where(wanted, ring[(first + number - 1) % n_pages], table))
    back = held & (column >= ((past + taken + page - 1) // page)[:, None])
    place = (first + count + back.flatten().cumsum(0).view(B, columns) - 1) % n_pages
    more = torch.cat((ring, ring[:1])).scatter_(0, torch.where(back, place, n_pages).flatten(), table.flatten())
    ring.copy_(more[:n_pages])
    table.masked_fill_(back, -1)
    used = wanted.sum()
    span.copy_(torch.stack(((first + used) % n_pages, count - used + back.sum())))
    row = torch.arange(rows, device=table.device)
    b = torch.searchsorted(end, row, right=True).clamp(max=B - 1)
    t = row - (end - new)[b]
    token = (row < end[-1]) & admitted[b]
    key = (past[b] + t).clamp(0, columns * page - 1)
    slots = torch.where(token, table[b, key // page].long() * page + key % page, -1).to(torch.int32)
    positions = torch.where(token, state["next_positions"][b] + t, -1).to(torch.int32)
    state["seq_lens"].copy_(past + taken)
    state["next_positions"].add_(taken)
    offsets = torch.cat((torch.zeros_like(end[:1]), end)).clamp(max=rows).to(torch.int32)
    return offsets, positions, slots, taken.to(torch.int32)


def _plain_rope(state):
    qkv, kv, n_q = state["qkv"], state["kv_pages"], state["q_heads"]
    Hkv, page = kv.shape[1] // 2, kv.shape[2]
    where = state["positions"].long().clamp(min=0)
    c, s = state["cos"][where][:, None], state["sin"][where][:, None]
    x = qkv[:, :n_q + Hkv].float()
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    x = torch.cat((lo * c - hi * s, hi * c + lo * s), -1).to(qkv.dtype)
    token = state["positions"] >= 0
    qkv[:, :n_q + Hkv] = torch.where(token[:, None, None], x, qkv[:, :n_q + Hkv])
    filed = token & (state["slots"] >= 0)
    slot = state["slots"][filed].long()
    at = (slot // page, slice(None), slot % page)
    kv[at] = qkv[filed][:, n_q:]
    state["weights"][at] = 0.0
    state["key_positions"][at] = state["positions"][filed][:, None].expand(-1, Hkv)


def _descent(parents):
    """[B, N, N]: whether token j is token i or what it descends from."""
    B, N = parents.shape
    up = torch.zeros((B, N, N + 1), device=parents.device)
    up.scatter_(2, torch.where(parents < 0, N, parents).long()[..., None], 1.0)
    up = up[..., :N].contiguous()
    seen = torch.eye(N, device=parents.device).expand(B, N, N)
    for _ in range(max(1, (N - 1).bit_length())):   # the paths of up to 1, 3, 7, .. steps
        seen, up = seen + torch.matmul(up, seen.contiguous()), torch.matmul(up, up.contiguous())
    return seen > 0.5


def _paged(x, table):
    """[n_pages, H, page, ...] -> [B, H, slots, ...]: the pages of every sequence one behind the other."""
    return x[table.long()].transpose(1, 2).flatten(2, 3)


def _plain_tree(state):
    q, kv, seq_lens = state["q"], state["kv_pages"], state["seq_lens"].long()
    B, Hq, N, _ = q.shape
    Hkv = kv.shape[1] // 2
    k, v = (_paged(kv[:, i * Hkv:(i + 1) * Hkv], state["block_table"]).float() for i in (0, 1))
    key = torch.arange(k.shape[2], device=q.device)
    new = torch.full_like(seq_lens, N) if state["new_lens"] is None else state["new_lens"].long()
    begin = (seq_lens - new)[:, None]
    drafted = (key >= begin) & (key < seq_lens[:, None])
    index = (key - begin).clamp(0, N - 1)
    seen = _descent(state["parents"]).gather(2, index[:, None].expand(B, N, -1))
    visible = (key < begin)[:, None] | (drafted[:, None] & seen)
    visible &= (torch.arange(N, device=q.device) < new[:, None])[..., None]
    o, lse = _attention(q.float(), k, v, visible)
    return o.to(q.dtype), lse


def _plain_keep(state):
    kv, table, path, new = state["kv_pages"], state["block_table"], state["path"].long(), state["new_lens"].long()
    page = kv.shape[2]
    goes_on = (path > torch.cat((torch.full_like(path[:, :1], -1), path[:, :-1]), 1)) & (path < new[:, None])
    on_path = goes_on.long().cumprod(1).bool()
    begin = state["seq_lens"].long() - new
    b, to = on_path.nonzero(as_tuple=True)
    src, dst = begin[b] + path[b, to], begin[b] + to
    sp, dp = table[b, src // page].long(), table[b, dst // page].long()
    kv[dp, :, dst % page] = kv[sp, :, src % page]
    if state["weights"] is not None:
        state["weights"][dp, :, dst % page] = state["weights"][sp, :, src % page]
        state["key_positions"][dp, :, dst % page] = state["key_positions"][sp, :, src % page]
    return (begin + on_path.sum(1)).to(torch.int32)


# ---- a pass --------------------------------------------------------------------------------------------------------


def _ops():
    package = os.path.abspath("understanding-gpu-architecture-implications-on-llm-serving-workloads_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import fmha_unified
    return fmha_unified.ops


def run(state):
    kind = state["kind"]
    if kind == "packed":
        if own:
            o, lse = _ops().fine_fmha_packed_with_lse(state["q"], state["k"], state["v"], state["offsets"], causal=state["causal"])
        else:
            o, lse = _plain_packed(state)
        return {"o": o, "lse": lse}
    if kind == "plan":
        state["now"].copy_(state["saved"])
        if own:
            got = _ops().fine_plan_packed(state["block_table"], state["seq_lens"], state["new_lens"], state["free_pages"], state["free_span"],
                                          state["page"], state["rows"], next_positions=state["next_positions"])
        else:
            got = _plain_plan(state)
        return dict(zip(("offsets", "positions", "slots", "taken"), got), now=state["now"])
    if kind == "rope":
        if own:
            _ops().fine_rope_packed(state["qkv"], state["kv_pages"], state["slots"], state["cos"], state["sin"], state["positions"],
                                    state["q_heads"], weights=state["weights"], key_positions=state["key_positions"], keep_keys=True)
        else:
            _plain_rope(state)
        return {name: state[name] for name in ("qkv", "kv_pages", "weights", "key_positions")}
    cache = (state["kv_pages"], state["block_table"], state["seq_lens"])
    if kind == "tree":
        if own:
            o, lse = _ops().fine_fmha_tree_with_lse(state["q"], *cache, state["parents"], new_lens=state["new_lens"])
        else:
            o, lse = _plain_tree(state)
        return {"o": o, "lse": lse}
    if own:
        lens = _ops().fine_keep_path(*cache, state["new_lens"], state["path"], weights=state["weights"], key_positions=state["key_positions"])
    else:
        lens = _plain_keep(state)
    account = {} if state["weights"] is None else {name: state[name] for name in ("weights", "key_positions")}
    return dict(account, seq_lens=lens, kv_pages=state["kv_pages"])


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def _exact_head(q, k, v, hidden):
    """One head: q [N, 128], k, v [S, 128], hidden [N, S] or None, all in 64 bits."""
    s = q @ k.T / D ** 0.5
    if hidden is not None:
        s = s.masked_fill_(hidden, float("-inf"))
    lse = s.logsumexp(-1)
    return s.softmax(-1).nan_to_num(0.0) @ v, lse


def _exact_plan(st):
    page, rows, new = st["page"], st["rows"], st["new_lens"].tolist()
    table, lens, ring = st["block_table"].tolist(), st["seq_lens"].tolist(), st["free_pages"].tolist()
    (first, count), texts = st["free_span"].tolist(), st["next_positions"].tolist()
    n_pages, columns = len(ring), len(table[0])
    free = [ring[(first + i) % n_pages] for i in range(count)]
    offsets, positions, slots, taken, came_back, need_so_far, used = [0], [-1] * rows, [-1] * rows, [], [], 0, 0
    for b, n in enumerate(new):
        at, have = offsets[-1], lens[b]
        offsets.append(min(at + n, rows))
        ok = at + n <= rows and have + n <= columns * page
        needed = [c for c in range(have // page, -(-(have + n) // page)) if not 0 <= table[b][c] < n_pages] if ok and n > 0 else []
        need_so_far += len(needed)
        ok = ok and (not needed or need_so_far <= count)
        taken.append(n if ok else 0)
        if ok:
            for c in needed:
                table[b][c] = free[used]
                used += 1
            for t in range(n):
                positions[at + t], slots[at + t] = texts[b] + t, table[b][(have + t) // page] * page + (have + t) % page
            lens[b], texts[b] = have + n, texts[b] + n
        for c in range(-(-lens[b] // page), columns):
            if 0 <= table[b][c] < n_pages:
                came_back.append(table[b][c])
                table[b][c] = -1
    for i, p in enumerate(came_back):
        ring[(first + count + i) % n_pages] = p
    now = sum(table, []) + lens + ring + [(first + used) % n_pages, count - used + len(came_back)] + texts
    return {name: torch.tensor(x, dtype=torch.int32) for name, x in
            dict(offsets=offsets, positions=positions, slots=slots, taken=taken, now=now).items()}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(st)
    Hkv, group = case["Hkv"], case.get("Hq", 0) // case["Hkv"]
    if case["kind"] == "packed":
        lens = _lengths(case["B"], case["longest"], case["ragged"])
        rows = sum(lens) + case["spare"]
        o = torch.zeros((rows, case["Hq"], D), device="cuda", dtype=torch.float64)
        lse = torch.full((case["Hq"], rows), float("-inf"), device="cuda", dtype=torch.float64)
        at = 0
        for n in lens:
            hidden = torch.ones((n, n), device="cuda", dtype=torch.bool).triu(1) if case["causal"] else None
            for h in range(case["Hq"]):
                part = [st[x][at:at + n, i].double() for x, i in (("q", h), ("k", h // group), ("v", h // group))]
                o[at:at + n, h], lse[h, at:at + n] = _exact_head(*part, hidden)
            at += n
        return {"o": o, "lse": lse}
    page = case["page"]
    if case["kind"] == "rope":
        n_q, tokens = case["Hq"], st["qkv"].shape[0] - case["spare"]
        qkv, pages, weights, positions = st["qkv"].double(), st["kv_pages"].double(), st["weights"].double(), st["key_positions"]
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"][:tokens].long()][:, None]
        y = torch.complex(qkv[:tokens, :n_q + Hkv, :D // 2], qkv[:tokens, :n_q + Hkv, D // 2:]) * turn
        qkv[:tokens, :n_q + Hkv] = torch.cat((y.real, y.imag), -1)
        pg, sl = st["slots"][:tokens].long() // page, st["slots"][:tokens].long() % page
        for h in range(2 * Hkv):
            pages[pg, h, sl] = qkv[:tokens, n_q + h]
        for h in range(Hkv):
            weights[pg, h, sl], positions[pg, h, sl] = 0.0, st["positions"][:tokens]
        return {"qkv": qkv, "kv_pages": pages, "weights": weights, "key_positions": positions}
    lens, new = _drafts(case)
    table = st["block_table"].long()

    def places(b, keys):
        keys = torch.as_tensor(keys, device="cuda", dtype=torch.long)
        return table[b][keys // page], keys % page

    if case["kind"] == "keep":
        left, paths = [], st["path"].tolist()
        for b in range(case["B"]):
            begin, accepted = lens[b] - new[b], []
            for i in paths[b]:
                if not (accepted[-1] if accepted else -1) < i < new[b]:
                    break
                accepted.append(i)
            for j, i in enumerate(accepted):
                (tp, ts), (fp, fs) = places(b, [begin + j]), places(b, [begin + i])
                for t in (st["kv_pages"], st["weights"], st["key_positions"]):
                    if t is not None:
                        t[tp, :, ts] = t[fp, :, fs]
            left.append(begin + len(accepted))
        account = {} if st["weights"] is None else {name: st[name] for name in ("weights", "key_positions")}
        return dict(account, seq_lens=torch.tensor(left, dtype=torch.int32), kv_pages=st["kv_pages"])
    q, parents = st["q"], st["parents"].tolist()
    o = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.full(q.shape[:3], float("-inf"), device="cuda", dtype=torch.float64)
    for b in range(case["B"]):
        hidden = [[True] * new[b] for _ in range(new[b])]
        for i in range(new[b]):
            j = i
            while j >= 0:
                hidden[i][j] = False
                j = parents[b][j]
        begin = lens[b] - new[b]
        hidden = torch.cat((torch.zeros((new[b], begin), dtype=torch.bool), torch.tensor(hidden)), 1).cuda()
        pg, sl = places(b, range(lens[b]))
        for h in range(case["Hq"]):
            k, v = (st["kv_pages"][pg, h // group + i * Hkv, sl].double() for i in (0, 1))
            o[b, h, :new[b]], lse[b, h, :new[b]] = _exact_head(q[b, h, :new[b]].double(), k, v, hidden)
    return {"o": o, "lse": lse}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "plan":
        past, new = _requests(case)
        # the table once, positions and slots of the tokens, lengths, offsets and positions of the sequences
        return {"bytes": 4 * case["B"] * case["columns"] + 8 * (sum(new) + case["spare"]) + 32 * case["B"], "flops": 0}
    Hkv, Hq = case["Hkv"], case.get("Hq", 0)
    if kind == "packed":
        lens = _lengths(case["B"], case["longest"], case["ragged"])
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (4 * D * (Hq + Hkv) + 4 * Hq) + case["spare"] * Hq * (2 * D + 4), "flops": 4 * D * Hq * pairs}
    if kind == "rope":
        tokens = sum(_lengths(case["B"], case["longest"], case["ragged"]))
        return {"bytes": tokens * (2 * D * (Hq + 2 * Hkv + Hq + 3 * Hkv) + 4 * D + 8 + 8 * Hkv), "flops": 6 * tokens * (Hq + Hkv) * D // 2}
    lens, new = _drafts(case)
    if kind == "keep":
        # a quarter of the drafted tokens at most, half of those on average, move: read and written
        moved = sum(-(-case["nodes"] // 4) / 2 for _ in new)
        return {"bytes": int(moved * Hkv * (8 * D + 16 * case["account"])) + 4 * case["B"] * (4 + -(-case["nodes"] // 4)), "flops": 0}
    rows = case["B"] * case["nodes"]
    pairs = sum(n * (t - n) + n * 8 for t, n in zip(lens, new))   # (a drafted token descends from a few)
    return {"bytes": 4 * D * Hkv * sum(lens) + rows * Hq * (4 * D + 4) + 4 * rows, "flops": 4 * D * Hq * pairs}
