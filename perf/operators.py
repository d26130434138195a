"""The operators of generation with drafted tokens over a paged KV cache, as timed cases.

Four operators that belong to one decoding step:

  tree_attention  attention of the nodes of a token tree over a paged cache; writes the nodes' keys and values
  verify_tree     walks the tree against the target's probabilities with given random numbers, draws the next token
  kv_commit       moves the accepted nodes' keys and values together and makes room for the next tree
  kv_fork         sequences take over, share or give up the pages of other sequences

`run` computes each in its plain form (elementary torch operations in 32 bits) or, with `own`, calls fxlm.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_FIX = float(2 ** 36)  # probabilities are summed as whole multiples of 2^-36


# ------------------------------------------------------------------ cases
def _attn(name, dtype, B, T, Hq, Hkv, D, ctx, page):
    c = {"op": "attn", "dtype": dtype, "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "ctx": ctx, "page": page}
    return dict(c, name=name) if name else c


def _verify(name, B, T, V, chain, draft):
    c = {"op": "verify", "B": B, "T": T, "V": V, "chain": chain, "draft": draft}
    return dict(c, name=name) if name else c


def _pages(name, op, dtype, S, T, L, H, D, page, ctx):
    c = {"op": op, "dtype": dtype, "S": S, "T": T, "L": L, "H": H, "D": D, "page": page, "ctx": ctx}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the next token of one sequence at the end of the GPT d768 model's 1024-token window, without a draft
        _attn("attn_one_token", "bf16", 1, 1, 12, 12, 64, 1023, 16),
        # the same model, eight sequences with trees of up to 16 drafted tokens, fp16
        _attn("attn_tree_d768", "f16", 8, 16, 12, 12, 64, 1008, 16),
        # a serving batch with shared key heads, a short draft per sequence, uneven lengths
        _attn("attn_batch_shared_heads", "bf16", 48, 4, 32, 8, 128, 8192, 64),
        # few sequences, wide trees, eight query heads a key head: the case with the most arithmetic
        _attn("attn_wide_tree", "bf16", 4, 63, 32, 4, 128, 12001, 128),
        # one long document of an odd length
        _attn("attn_one_long", "bf16", 1, 8, 32, 8, 128, 100003, 32),
        # the 32-bit parity mode, odd lengths
        _attn("attn_f32", "f32", 3, 5, 12, 12, 64, 517, 32),
        # one sequence, a chain without draft probabilities (drafts looked up, not sampled), the model's vocabulary
        _verify("verify_one_chain", 1, 8, 32768, True, False),
        # a serving batch of trees drawn from a draft model, odd vocabulary
        _verify("verify_batch_tree", 64, 32, 50257, False, True),
        # the end of one sequence's step on the GPT d768 model
        _pages("commit_one", "commit", "bf16", 1, 8, 12, 12, 64, 16, 500),
        # the end of a batch's step, wide trees, 32 layers
        _pages("commit_batch", "commit", "bf16", 64, 64, 32, 8, 128, 64, 150),
        # several samples of one prompt on the GPT d768 model
        _pages("fork_samples", "fork", "f16", 4, 1, 12, 12, 64, 16, 500),
        # a batch of beams, 32 layers
        _pages("fork_beams", "fork", "bf16", 48, 1, 32, 8, 128, 64, 250),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "verify", "commit", "fork"])
    if op == "attn":
        dt = rng.choice(["bf16", "bf16", "f16", "f32"])
        D = rng.choice([64, 128])
        G = rng.choice([1, 1, 2, 3, 4, 8])
        Hkv = _log(rng, 1, 16)
        B, T = _log(rng, 1, 64), _log(rng, 1, 64)
        ctx = _log(rng, 1, 100000)
        # no more bytes than attn_batch_shared_heads, no more products than attn_wide_tree
        most = (330e6 if dt != "f32" else 40e6) / (B * Hkv * D)
        ctx = int(min(ctx, max(1, most), max(1, (10e9 if dt != "f32" else 1e9) / (B * Hkv * G * T * D))))
        return _attn(None, dt, B, T, Hkv * G, Hkv, D, ctx, rng.choice([16, 32, 64, 128]))
    if op == "verify":
        V = _log(rng, 256, 131072)
        B, T = _log(rng, 1, 64), _log(rng, 1, 64)
        while B * T * V > 64 * 32 * 50257:
            B, T = max(1, B // 2), max(1, T - T // 3)
        return _verify(None, B, T, V, rng.random() < 0.3, rng.random() < 0.6)
    dt = rng.choice(["bf16", "f16", "f32"])
    D, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    S, L, H = _log(rng, 1 if op == "commit" else 2, 48), _log(rng, 1, 32), _log(rng, 1, 12)
    T, ctx = (_log(rng, 1, 64) if op == "commit" else 1), _log(rng, 1, 300)
    while S * ((ctx + 2 * T) // page + 3) * page * L * H * D * _SIZE[dt] > 1.2e9:
        S, L = max(2, S // 2), max(1, L - L // 3)
        ctx = max(1, ctx // 2)
    return _pages(None, op, dt, S, T, L, H, D, page, ctx)


# sizes that follow from the case alone
def _lens(n, ctx):
    return [ctx - (b * 7919) % (ctx // 2 + 1) for b in range(n)]


def _nodes(c):
    n = [c["T"] - (b * 3) % (c["T"] // 2 + 1) for b in range(c["B"])]
    if c["B"] >= 8:
        n[-1] = 0  # a slot that sits this step out
    return n


def _depths(c):
    return [1 + (s * 5 + 3) % min(c["T"], 9) for s in range(c["S"])]


def _path(T, d):
    return [i + (i * (T - d)) // max(d - 1, 1) for i in range(d)]


def _parents_of_slots(c):
    S = c["S"]
    return [-1 if s % 3 == 2 and s % 5 == 4 else s - s % 3 for s in range(S)]


def work(case):
    c = case
    if c["op"] == "attn":
        lens, n, e = _lens(c["B"], c["ctx"]), _nodes(c), _SIZE[c["dtype"]]
        row = c["D"] * e
        kv = sum(l for l, k in zip(lens, n) if k) * c["Hkv"] * row * 2
        new = sum(n) * c["Hkv"] * row * 2 * 2  # the nodes' keys and values, read and written
        q = sum(n) * c["Hq"] * row + c["B"] * c["T"] * c["Hq"] * row
        table = sum(-(-l // c["page"]) for l in lens) * 4
        flops = sum(4.0 * k * c["Hq"] * c["D"] * (l + (k + 1) / 2) for l, k in zip(lens, n))
        return {"bytes": kv + new + q + table, "flops": flops}
    if c["op"] == "verify":
        # the tree and a few values of each node, and the rows of one node: where the walk ends
        rows = 2 if c["draft"] else 1
        return {"bytes": c["B"] * (c["V"] * 4 * rows + c["T"] * (8 + 4 + 4 + 4 * rows + 4) + 12), "flops": c["B"] * c["V"] * 3.0}
    e, W = _SIZE[c["dtype"]], _width(c)
    token = c["L"] * 2 * c["H"] * c["D"] * e
    if c["op"] == "commit":
        moved = sum(sum(p != i for i, p in enumerate(_path(c["T"], d))) for d in _depths(c))
        return {"bytes": moved * token * 2 + c["S"] * (c["T"] * 4 + 24), "flops": 0}
    lens, par = _lens(c["S"], c["ctx"]), _parents_of_slots(c)
    copied = sum(lens[p] % c["page"] for s, p in enumerate(par) if p >= 0 and p != s)
    return {"bytes": copied * token * 2 + 2 * c["S"] * W * 4, "flops": 0}


def _width(c):
    """Entries of a row of the page table: room for the longest sequence and its next tree."""
    return -(-(c["ctx"] + 3 * c["T"]) // c["page"]) + 1


# ------------------------------------------------------------------ inputs
def _trees(B, T, chain, rng):
    """Parents of the nodes (node 0: the last committed token, -1) and, as 64-bit masks, what each node sees."""
    par = np.full((B, T), -1, np.int32)
    seen = np.zeros((B, T), np.uint64)
    for b in range(B):
        seen[b, 0] = 1
        for i in range(1, T):
            p = i - 1 if chain else int(rng.randint(max(0, i - 5), i))
            par[b, i] = p
            seen[b, i] = seen[b, p] | np.uint64(1 << i)
    return torch.from_numpy(par).cuda(), torch.from_numpy(seen.view(np.int64)).cuda()


def _table(held, W, P, rng):
    """Pages in a shuffled order, as after long use: table (-1 where nothing is held) and reference counts."""
    order = rng.permutation(P)[: int(sum(held))]
    table, at = np.full((len(held), W), -1, np.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    ref = np.zeros(P, np.int32)
    ref[order] = 1
    return torch.from_numpy(table).cuda(), torch.from_numpy(ref).cuda()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    rng = np.random.RandomState(seed % (2 ** 31))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = dict(c)
    if c["op"] == "attn":
        B, T, D, dt = c["B"], c["T"], c["D"], _DT[c["dtype"]]
        lens, n, W = _lens(B, c["ctx"]), _nodes(c), _width(c)
        held = [-(-(l + T) // c["page"]) for l in lens]
        P = sum(held) + max(2, sum(held) // 16)
        s["table"], _ = _table(held, W, P, rng)
        s["k_pages"], s["v_pages"] = (randn(P, c["Hkv"], c["page"], D, dtype=dt) for _ in range(2))
        # q, k and v as one projection leaves them
        qkv = (randn(B, T, c["Hq"] + 2 * c["Hkv"], D) * 1.5).to(dt)
        s["q"], s["k"], s["v"] = qkv.split([c["Hq"], c["Hkv"], c["Hkv"]], dim=2)
        _, s["mask"] = _trees(B, T, False, rng)
        s["lens"], s["n"] = _i32(lens), _i32(n)
        return s
    if c["op"] == "verify":
        B, T, V = c["B"], c["T"], c["V"]
        s["parents"], _ = _trees(B, T, c["chain"], rng)
        logits = randn(B, T, V) * 3
        s["p"] = torch.softmax(logits, -1)
        s["q"] = torch.softmax(logits.mul_(0.85) + randn(B, T, V), -1) if c["draft"] else None
        del logits
        src = s["q"] if c["draft"] else s["p"]
        s["tokens"] = torch.empty(B, T, dtype=torch.int64, device="cuda")
        rows = torch.arange(B, device="cuda")
        for i in range(T):  # each node drawn from its parent's row
            w = src[rows, s["parents"][:, i].clamp(min=0).long()]
            e = torch.empty(B, V, device="cuda").exponential_(generator=g)
            s["tokens"][:, i] = (w / e).argmax(-1)
        s["n"] = _i32(_nodes(c))
        s["u"] = torch.rand(B, T, generator=g, device="cuda")
        return s
    S, L, H, D, T, page, dt = c["S"], c["L"], c["H"], c["D"], c["T"], c["page"], _DT[c["dtype"]]
    lens, W = _lens(S, c["ctx"]), _width(c)
    held = [-(-(l + (T if c["op"] == "commit" else 0)) // page) for l in lens]
    P = sum(held) + S * (-(-T // page) + 1) + 3
    s["table"], s["ref"] = _table(held, W, P, rng)
    s["k"], s["v"] = (randn(L, P, H, page, D, dtype=dt) for _ in range(2))
    s["lens"], s["n_pages"] = _i32(lens), _i32(held)
    if c["op"] == "commit":
        depth = _depths(c)
        s["path"] = _i32([(_path(T, d) + [-1] * T)[:T] for d in depth])
        s["n_path"], s["room"] = _i32(depth), _i32([T] * S)
    else:
        s["parents"] = _i32(_parents_of_slots(c))
    return s


# ------------------------------------------------------------------ plain forms
def _plain_attn(s):
    B, T, Hq, D = s["q"].shape
    Hkv, page, W = s["Hkv"], s["page"], s["table"].shape[1]
    lens, n, table = s["lens"].long(), s["n"].long(), s["table"].long()
    t = torch.arange(T, device="cuda")
    live = t[None] < n[:, None]                                          # (B, T)
    # the nodes' keys and values go into the slots after the sequence
    at = lens[:, None] + t[None]
    pg, off = table.gather(1, at // page), at % page
    for pool, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])):
        pool[pg, :, off] = torch.where(live[..., None, None], new, pool[pg, :, off])
    # keys and values of the context, then of the nodes: (B, Hkv, N, D) in 32 bits
    N = W * page
    ctx = [p[table.clamp(min=0)].float().transpose(1, 2).reshape(B, Hkv, N, D) for p in (s["k_pages"], s["v_pages"])]
    k = torch.cat([ctx[0], s["k"].float().transpose(1, 2)], 2)
    v = torch.cat([ctx[1], s["v"].float().transpose(1, 2)], 2)
    del ctx
    in_ctx = torch.arange(N, device="cuda")[None] < lens[:, None]        # (B, N)
    in_tree = ((s["mask"][..., None] >> t) & 1).bool() & live[:, None]   # (B, T, T)
    see = torch.cat([in_ctx[:, None].expand(B, T, N), in_tree], 2) & live[..., None]
    G = Hq // Hkv
    q = s["q"].float().view(B, T, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * T, D)
    x = (q @ k.transpose(2, 3)).view(B, Hkv, G, T, -1) / math.sqrt(D)
    x = torch.where(see[:, None, None], x, float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), 0.0, m))
    z = e.sum(-1, keepdim=True)
    v = torch.where(torch.cat([in_ctx, live], 1)[:, None, :, None], v, 0.0)
    o = (e.view(B, Hkv, G * T, -1) @ v).view(B, Hkv, G, T, D) / torch.where(z == 0, 1.0, z)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype), s["k_pages"], s["v_pages"]


def _fixed(w):
    return (torch.where(w > 0, w, 0.0).clamp(max=1.0) * _FIX).to(torch.int64)


def _plain_verify(s):
    p, q, tokens, par, n, u = s["p"], s["q"], s["tokens"], s["parents"], s["n"], s["u"]
    B, T, V = p.shape
    rows = torch.arange(B, device="cuda")
    cur = torch.zeros(B, dtype=torch.int64, device="cuda")
    path = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = torch.where(n > 0, 0, -1)
    n_path = (n > 0).to(torch.int32)
    w = p[:, 0].clone()                                 # what is left of the current node's row
    scale = torch.ones(B, device="cuda")                # its probabilities are w * scale (with q), w / mass (without)
    mass = torch.ones(B, device="cuda")
    empty = torch.zeros(B, dtype=torch.bool, device="cuda")
    # a node's index is above its parent's: one sweep in index order meets the children of each node the walk reaches
    for c in range(1, T):
        x = tokens[:, c]
        inside = (x >= 0) & (x < V)
        xi = x.clamp(0, V - 1)
        test = (par[:, c] == cur) & (c < n) & ~empty
        a = w[rows, xi]
        a = torch.where(inside & (a > 0), a, 0.0)
        if q is None:
            a = a.clamp(max=1.0)
            take = test & (u[:, c] * mass < a)
        else:
            take = test & (u[:, c] * torch.where(inside, q[rows, cur, xi], 0.0) < a * scale)
        drop = test & ~take
        if q is None:
            mass = torch.where(drop, (mass - a).clamp(min=0.0), mass)
            w[rows, xi] = torch.where(drop & inside, 0.0, w[rows, xi])
        else:
            r = w * scale[:, None] - q[rows, cur]
            r = torch.where(r > 0, r, 0.0)
            total = _fixed(r).sum(-1)
            empty = empty | (drop & (total == 0))
            w = torch.where(drop[:, None], r, w)
            scale = torch.where(drop, 1.0 / (total.float() * (1.0 / _FIX)), scale)
        cur = torch.where(take, c, cur)
        w = torch.where(take[:, None], p[:, c], w)
        scale, mass = torch.where(take, 1.0, scale), torch.where(take, 1.0, mass)
        path[rows, n_path.long().clamp(max=T - 1)] = torch.where(take, c, path[rows, n_path.long().clamp(max=T - 1)]).int()
        n_path = n_path + take.int()
    # the next token: what is left of the last node's row, or the row itself where nothing is left
    f = _fixed(w)
    f = torch.where((f.sum(-1) == 0)[:, None], _fixed(p[rows, cur]), f)
    cum = f.cumsum(-1)
    k = (u[:, 0] * 16777216.0).to(torch.int64).clamp(0, 16777215)
    nxt = (cum <= ((cum[:, -1] * k) >> 24)[:, None]).sum(-1)
    nxt = torch.where((cum[:, -1] > 0) & (n > 0), nxt, -1)
    return path, n_path, nxt


def _grow(table, n_pages, ref, need):
    """Pages for every slot up to need[s], the lowest-numbered free ones in the order of the slots; none at all if they do not suffice."""
    free = ref == 0
    first = torch.argsort((~free).to(torch.int8), stable=True)
    j = torch.arange(table.shape[1], device="cuda")[None]
    want = (j >= n_pages[:, None]) & (j < need[:, None])
    total = want.sum()
    ok = total <= free.sum()
    rank = (want.reshape(-1).cumsum(0) - 1).view_as(want).clamp(0, ref.numel() - 1)
    table.copy_(torch.where(want & ok, first[rank].int(), table))
    n_pages.copy_(torch.where(ok, torch.maximum(need, n_pages), n_pages))
    ref.add_((free & (free.cumsum(0) <= torch.where(ok, total, 0))).int())


def _plain_commit(s):
    table, page = s["table"], s["page"]
    S, T = s["path"].shape
    i = torch.arange(T, device="cuda")[None]
    live = i < s["n_path"][:, None]
    dst = s["lens"].long()[:, None] + i
    src = s["lens"].long()[:, None] + torch.where(live, s["path"].long(), i)
    dp, do, sp, so = table.long().gather(1, dst // page), dst % page, table.long().gather(1, src // page), src % page
    for pool in (s["k"], s["v"]):
        pool[:, dp, :, do] = pool[:, sp, :, so]
    lens = s["lens"] + s["n_path"]
    need = torch.where(s["room"] > 0, ((lens + s["room"] + page - 1) // page).clamp(max=table.shape[1]), 0).int()
    _grow(table, s["n_pages"], s["ref"], need)
    return lens, table, s["n_pages"], s["ref"], s["k"], s["v"]


def _plain_fork(s):
    table, ref, lens, page, n_pages, par = s["table"], s["ref"], s["lens"], s["page"], s["n_pages"], s["parents"].long()
    S, W = table.shape
    slot = torch.arange(S, device="cuda")
    p = par.clamp(min=0)
    held = torch.where(par >= 0, lens[p], 0)
    count = (held + page - 1) // page
    # a partly filled last page stays with one heir: the slot itself, else the first that forks from it; the others copy it
    kids = par[None] == slot[:, None]                                    # (from, to)
    first = torch.where(kids.any(1), kids.int().argmax(1), -1)
    heir = torch.where(par == slot, slot, first)
    copy = (held % page > 0) & (heir[p] != slot)
    free = ref == 0
    order = torch.argsort((~free).to(torch.int8), stable=True)
    ok = copy.sum() <= free.sum()
    new = order[(copy.long().cumsum(0) - 1).clamp(0, ref.numel() - 1)]
    j = torch.arange(W, device="cuda")[None]
    last = (count - 1).clamp(min=0)
    t = torch.where(j < count[:, None], table[p], -1)
    old_tail = t.gather(1, last[:, None].long())[:, 0].long()
    old_tail = torch.where(old_tail >= 0, old_tail, ref.argmax())  # a page in use, so none of `new`
    t = torch.where(copy[:, None] & (j == last[:, None]), new[:, None].int(), t)
    # the copies: `held % page` tokens of the old last page into the new one, in every layer
    dst = torch.where(copy & ok, new, old_tail)
    keep = torch.arange(page, device="cuda")[None] < (held % page)[:, None]
    for pool in (s["k"], s["v"]):
        moved = torch.where((keep & (copy & ok)[:, None])[None, :, None, :, None], pool[:, old_tail], pool[:, dst])
        pool.index_copy_(1, dst, moved)
    was, now = (j < n_pages[:, None]).int(), (j < count[:, None]).int()
    delta = torch.zeros_like(ref).index_add_(0, table.clamp(min=0).reshape(-1).long(), -was.reshape(-1))
    delta.index_add_(0, t.clamp(min=0).reshape(-1).long(), now.reshape(-1))
    ref.add_(torch.where(ok, delta, 0))
    table.copy_(torch.where(ok, t, table))
    n_pages.copy_(torch.where(ok, count.int(), n_pages))
    lens.copy_(torch.where(ok, held.int(), lens))
    return table, n_pages, lens, ref, s["k"], s["v"]


def run(state):
    s = state
    if own:
        f = _fxlm()
        if s["op"] == "attn":
            o = f.tree_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["n"], s["mask"])
            return o, s["k_pages"], s["v_pages"]
        if s["op"] == "verify":
            return f.verify_tree(s["tokens"], s["parents"], s["n"], s["p"], s["u"], draft_probs=s["q"])
        if s["op"] == "commit":
            lens = f.kv_commit(s["k"], s["v"], s["table"], s["n_pages"], s["lens"], s["ref"], s["path"], s["n_path"], room=s["room"])
            return lens, s["table"], s["n_pages"], s["ref"], s["k"], s["v"]
        f.kv_fork(s["k"], s["v"], s["table"], s["n_pages"], s["lens"], s["ref"], s["parents"])
        return s["table"], s["n_pages"], s["lens"], s["ref"], s["k"], s["v"]
    return {"attn": _plain_attn, "verify": _plain_verify, "commit": _plain_commit, "fork": _plain_fork}[s["op"]](s)


def _fxlm():
    if "fxlm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "radeon-igpu-forge_b200"))
        import fxlm  # noqa: F401
    return sys.modules["fxlm"]


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """From the definitions, one sequence and one node (or page) at a time. The verification gives whole numbers only."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    return {"attn": _exact_attn, "commit": _exact_commit, "fork": _exact_fork}[case["op"]](s)


def _exact_attn(s):
    B, T, Hq, D = s["q"].shape
    page, G = s["page"], Hq // s["Hkv"]
    kp, vp = s["k_pages"], s["v_pages"]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    table, lens, n = s["table"].tolist(), s["lens"].tolist(), s["n"].tolist()
    for b in range(B):
        pages = torch.tensor(table[b][: -(-lens[b] // page)], device="cuda", dtype=torch.int64)
        seen = [[j for j in range(n[b]) if (m >> j) & 1] for m in s["mask"][b].tolist()]
        for h in range(s["Hkv"]):
            k, v = (x[pages, h].reshape(-1, D)[: lens[b]].double() for x in (kp, vp))
            nk, nv = s["k"][b, :, h].double(), s["v"][b, :, h].double()
            qs = s["q"][b, :, h * G:(h + 1) * G].double()
            for i in range(n[b]):
                kk, vv = torch.cat([k, nk[seen[i]]]), torch.cat([v, nv[seen[i]]])
                if len(kk):
                    out[b, i, h * G:(h + 1) * G] = torch.softmax(qs[i] @ kk.T / math.sqrt(D), -1) @ vv
        for i in range(n[b]):
            at = lens[b] + i
            kp[table[b][at // page], :, at % page] = s["k"][b, i]
            vp[table[b][at // page], :, at % page] = s["v"][b, i]
    return out, kp.double(), vp.double()


def _exact_commit(s):
    page = s["page"]
    table, lens, path, n = (s[k].tolist() for k in ("table", "lens", "path", "n_path"))
    for b in range(len(lens)):
        for i in range(n[b]):
            src, dst = lens[b] + path[b][i], lens[b] + i
            for pool in (s["k"], s["v"]):
                pool[:, table[b][dst // page], :, dst % page] = pool[:, table[b][src // page], :, src % page]
    return None, None, None, None, s["k"].double(), s["v"].double()


def _exact_fork(s):
    page = s["page"]
    table, lens, ref, par = (s[k].tolist() for k in ("table", "lens", "ref", "parents"))
    free = iter([i for i, r in enumerate(ref) if r == 0])
    taken = set(i for i, p in enumerate(par) if p == i)
    for i, p in enumerate(par):
        if p < 0 or p == i or lens[p] % page == 0:
            continue
        if p not in taken:
            taken.add(p)
            continue
        new, old = next(free), table[p][lens[p] // page]
        for pool in (s["k"], s["v"]):
            pool[:, new, :, : lens[p] % page] = pool[:, old, :, : lens[p] % page]
    return None, None, None, None, s["k"].double(), s["v"].double()


if __name__ == "__main__":
    for one in listed() + [draw(random.Random(i)) for i in range(12)]:
        print(one, work(one))
