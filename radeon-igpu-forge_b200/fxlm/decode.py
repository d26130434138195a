"""fxlm.decode: generation with a paged KV cache and drafted tokens.

The reference's sampler re-runs the window for every token
(ml/fxlm/sample.py:63-73). `generate_cached` draws from the same distribution
(temperature and top-k as there) but keeps the keys and values of the sequence
in a PagedKVCache: each step runs the model on the nodes of a token tree, the
last token and what follows it elsewhere in the sequence (`draft_from_text`),
keeps the longest accepted path and draws the next token behind it. With
`draft=0` the tree is the last token alone. Several samples of one prompt share
the prompt's pages (kv_fork).

The model's positions are absolute (pos_emb has seq_len rows), so a cache holds
up to seq_len tokens; past that `generate_cached` goes on with the reference's
loop on the last seq_len tokens.
"""
import torch

from fxb200 import _lib, ops
from .linear import fused_linear, fused_mlp
from .norm import rms_norm
from .paged import MAX_NODES, kv_commit, kv_fork, kv_reserve, tree_attention
from .speculate import verify_tree


class PagedKVCache:
    """Keys and values of `slots` sequences in pages of one pool for all layers.

    k, v (L, P, H, page, D); page_table (slots, W), n_pages, lens (slots,), ref
    (P,): see fxlm.paged. `pages` defaults to what every slot needs for
    `max_len` tokens.
    """

    def __init__(self, n_layer, n_head, head_dim, slots, max_len, device, dtype, page=16, pages=None):
        W = -(-max_len // page)
        P = slots * W if pages is None else pages
        both = torch.zeros(n_layer, P, 2, n_head, page, head_dim, device=device, dtype=dtype)
        self.k, self.v = both[:, :, 0], both[:, :, 1]
        self.page, self.slots, self.max_len = page, slots, max_len
        i32 = dict(device=device, dtype=torch.int32)
        self.page_table = torch.full((slots, W), -1, **i32)
        self.n_pages, self.lens, self.ref = torch.zeros(slots, **i32), torch.zeros(slots, **i32), torch.zeros(P, **i32)

    def reserve(self, room):
        """Pages for room[s] (slots,) int32 more tokens of every slot."""
        kv_reserve(self.page_table, self.n_pages, self.lens, self.ref, room, self.page)

    def commit(self, path, n_path, room=None):
        """Keep the nodes path[s, :n_path[s]] of the last tree, make room for the next one."""
        self.lens.copy_(kv_commit(self.k, self.v, self.page_table, self.n_pages, self.lens, self.ref, path, n_path,
                                  room=room))

    def fork(self, parents):
        """Slot s takes over the sequence of slot parents[s] (-1: it is emptied)."""
        kv_fork(self.k, self.v, self.page_table, self.n_pages, self.lens, self.ref, parents)

    def check(self):
        """Synchronise and raise RuntimeError if a call since the last check did not fit the pool."""
        _lib.raise_on_device_error("in a KV cache")


def tree_logits(model, cache, tokens, n_nodes, mask, depth):
    """Logits (S, T, V) of a fxlm.GPT after each node of token trees that
    continue the sequences of `cache`: tokens, mask, depth (S, T) int64 (what
    each node sees, see tree_masks, and its distance from the root), n_nodes
    (S,) int32. Writes the nodes' keys and values behind the sequences
    (cache.reserve first). Not differentiable: call it under torch.no_grad()."""
    cfg = model.cfg
    if cfg.linear_impl != "fused":
        raise ValueError("tree_logits needs linear_impl='fused'")
    S, T = tokens.shape
    D, H = cfg.d_model, cfg.n_head
    w = model.tok_emb.weight
    x = torch.empty(S, T, D, device=w.device, dtype=w.dtype)
    rows = model.pos_emb[(cache.lens[:, None] + depth).clamp(0, cfg.seq_len - 1).reshape(-1)]
    _lib.call("fxb_embedding_fwd", _lib.dtype_code(w.dtype), _lib.ptr(tokens), _lib.ptr(w), _lib.ptr(rows),
              _lib.ptr(x), 1, S * T, D, w.shape[0], _lib.stream_ptr(w.device))
    for layer, blk in enumerate(model.blocks):
        qkv = fused_linear(rms_norm(x, blk.ln1_w, cfg.eps), blk.qkv.weight).view(S, T, 3, H, D // H)
        o = tree_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], cache.k[layer], cache.v[layer],
                           cache.page_table, cache.lens, n_nodes, mask)
        x = fused_linear(o.view(S, T, D), blk.proj.weight, residual=x)
        x = fused_mlp(rms_norm(x, blk.ln2_w, cfg.eps), blk.fc.weight, blk.fc2.weight, residual=x)
    return fused_linear(rms_norm(x, model.lnf_w, cfg.eps), model._head_w())


def _pack(trees, T):
    """(S, 5, T) int64 on the host: tokens, parents, masks, depths and, repeated,
    the number of nodes of each tree (tokens, parents); an empty list is a slot
    that sits out."""
    rows = []
    for tok, par in trees:
        mask, depth = [], []
        for i, p in enumerate(par):
            mask.append((mask[p] if i else 0) | 1 << i)
            depth.append(depth[p] + 1 if i else 0)
        pad = [0] * (T - len(tok))
        rows.append([tok + pad, par + [-1] * len(pad), [m - (1 << 64) if m >> 63 else m for m in mask] + pad,
                     depth + pad, [len(tok)] * T])
    return torch.tensor(rows)


def _unpack(x):
    return (x[:, 0].contiguous(), x[:, 1].int().contiguous(), x[:, 4, 0].int().contiguous(), x[:, 2].contiguous(),
            x[:, 3])


def tree_batch(trees, device):
    """(tokens, parents, n_nodes, mask, depth) on `device` from lists (tokens,
    parents), one a slot; an empty list is a slot that sits out."""
    return _unpack(_pack(trees, max(1, max(len(t) for t, _ in trees))).to(device))


class DecodeStep:
    """One decoding step of a batch: room for the trees, the model on their
    nodes, verification, commit. Nothing in it waits for the host, so from its
    third call on it is a captured CUDA graph (the first two set up what
    launches lazily); trees have up to `nodes` tokens."""

    def __init__(self, model, cache, nodes, temperature, top_k):
        dev = cache.lens.device
        self.model, self.cache, self.T = model, cache, nodes
        self.temperature, self.top_k = temperature, top_k
        self.x = torch.zeros(cache.slots, 5, nodes, device=dev, dtype=torch.int64)
        self.u = torch.zeros(cache.slots, nodes, device=dev)
        self.calls, self.graph, self.out, self._ws = 0, None, None, {}

    @torch.no_grad()
    def _run(self):
        tokens, parents, n, mask, depth = _unpack(self.x)
        self.cache.reserve(n)
        logits = tree_logits(self.model, self.cache, tokens, n, mask, depth)
        path, n_path, nxt = verify_tree(tokens, parents, n, next_probs(logits, self.temperature, self.top_k), self.u)
        self.cache.commit(path, n_path)
        return torch.cat([path.long(), n_path[:, None].long(), nxt[:, None]], 1)

    def __call__(self, trees, u):
        """Accepted node indices and the next token of every slot: a list of
        (path, next), ([], -1) where the tree is empty; next is -1 too where the
        model's probabilities are (NaN logits). u (slots, nodes) fp32."""
        self.x.copy_(_pack(trees, self.T))
        self.u.copy_(u)
        self.calls += 1
        if self.calls <= 2:
            out = self._run()
        else:
            if self.graph is None:
                self.graph = torch.cuda.CUDAGraph()
                with ops.graph_workspaces(self._ws), torch.cuda.graph(self.graph):
                    self.out = self._run()
            self.graph.replay()
            out = self.out
        return [(r[:r[-2]], r[-1]) for r in out.tolist()]


def draft_from_text(seq, nodes, ngram=3, width=2):
    """Tree of up to `nodes` tokens: the last token of `seq` (a list) and, below
    it, what followed the latest earlier occurrences of its last tokens (the
    longest n-gram that occurred, at most `ngram`; up to `width` of them, common
    beginnings merged). Returns (tokens, parents)."""
    tokens, parents = [seq[-1]], [-1]
    for n in range(min(ngram, len(seq) - 1), 0, -1):
        tail, found = seq[-n:], []
        for i in range(len(seq) - n - 1, -1, -1):
            if seq[i:i + n] == tail:
                found.append(i + n)
                if len(found) == width:
                    break
        if not found:
            continue
        for at in found:
            cur = 0
            for t in seq[at:at + max(1, (nodes - 1) // len(found))]:
                kid = next((c for c in range(cur + 1, len(tokens)) if parents[c] == cur and tokens[c] == t), None)
                if kid is None:
                    if len(tokens) == nodes:
                        break
                    tokens.append(t)
                    parents.append(cur)
                    kid = len(tokens) - 1
                cur = kid
        break
    return tokens, parents


def next_probs(logits, temperature, top_k):
    """The sampler's distribution (ml/fxlm/sample.py:66-72): fp32 softmax of the
    tempered logits, all but the top_k set to 0 (ties with the k-th kept)."""
    logits = logits.float() / max(temperature, 1e-5)
    if top_k > 0:
        kth = torch.topk(logits, min(top_k, logits.shape[-1])).values[..., -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    return torch.softmax(logits, dim=-1)


@torch.inference_mode()
def generate_cached(model, ids, max_new, temperature=0.8, top_k=50, generator=None, draft=7, samples=1, page=16,
                    stats=None):
    """Append max_new sampled tokens to `ids` (1-D or (1, n) int64); returns
    (samples, n + max_new). Each step verifies up to `draft` drafted tokens per
    sample (0: plain decoding). `stats`, a dict, receives the number of model
    steps and of tokens they gave."""
    seq_len, dev = model.cfg.seq_len, model.tok_emb.weight.device
    if not 0 <= draft < MAX_NODES:
        raise ValueError(f"draft={draft}: 0 to {MAX_NODES - 1}")
    if samples < 1 or ids.numel() < 1:
        raise ValueError("generate_cached: at least one sample and one token")
    prompt = ids.reshape(-1).tolist()
    n0, goal = len(prompt), len(prompt) + max_new
    seqs = [list(prompt) for _ in range(samples)]
    i32 = dict(device=dev, dtype=torch.int32)
    steps = given = 0
    if n0 <= seq_len and max_new > 0:
        cfg = model.cfg
        cache = PagedKVCache(cfg.n_layer, cfg.n_head, cfg.d_model // cfg.n_head, samples, seq_len + MAX_NODES, dev,
                             model.tok_emb.weight.dtype, page)
        # the prompt but for its last token, as chains of nodes in slot 0
        for at in range(0, n0 - 1, MAX_NODES):
            part = prompt[at:min(n0 - 1, at + MAX_NODES)]
            chain = (part, list(range(-1, len(part) - 1)))
            tokens, parents, n, mask, depth = tree_batch([chain] + [([], [])] * (samples - 1), dev)
            cache.reserve(n)
            tree_logits(model, cache, tokens, n, mask, depth)
            cache.commit((parents + 1).contiguous(), n)
        if samples > 1:
            cache.fork(torch.zeros(samples, **i32))  # every sample continues the prompt
        step = DecodeStep(model, cache, draft + 1, temperature, top_k)
        while any(len(s) < min(goal, seq_len + 1) for s in seqs):
            # len(s) - 1 tokens are committed, a tree starts with the last one; every node needs a position
            trees = [draft_from_text(s, min(draft, goal - len(s) - 1, seq_len - len(s)) + 1)
                     if len(s) < min(goal, seq_len + 1) else ([], []) for s in seqs]
            u = torch.rand(samples, draft + 1, device=dev, generator=generator)
            for s, (t, _), (path, nxt) in zip(seqs, trees, step(trees, u)):
                if path:
                    if nxt < 0:
                        cache.check()
                        raise RuntimeError("generate_cached: the model's probabilities of the next token are empty "
                                           "(NaN or infinite logits)")
                    s.extend([t[i] for i in path[1:]] + [nxt])
                    given += len(path)
            steps += 1
        cache.check()
    if stats is not None:
        stats.update(steps=steps, tokens=given)
    out = [torch.tensor(s[:goal], device=dev) for s in seqs]
    if any(len(x) < goal for x in out):
        from .sample import generate
        out = [generate(model, x, goal - len(x), temperature, top_k, generator)[0] for x in out]
    return torch.stack(out)
