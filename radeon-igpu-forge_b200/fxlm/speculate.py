"""fxlm.speculate: verification of drafted tokens against the target's probabilities."""
import torch

from .paged import MAX_NODES, _failed, _native, _refuse_devices, _refuse_i32


def _refuse(tokens, parents, n_nodes, target_probs, u, draft_probs):
    if tokens.dim() != 2:
        raise ValueError(f"tokens must be (B,T), got {tuple(tokens.shape)}")
    B, T = tokens.shape
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"T={T}: 1 to {MAX_NODES} nodes")
    if tokens.dtype != torch.int64 or not tokens.is_cuda:
        raise TypeError("tokens must be a cuda int64 tensor")
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    shape = (B, T, target_probs.shape[-1])
    for t, name in ((target_probs, "target_probs"), (draft_probs, "draft_probs")):
        if t is None:
            continue
        if t.dtype != torch.float32 or not t.is_cuda:
            raise TypeError(f"{name} must be a cuda fp32 tensor, got {t.dtype} on {t.device}")
        if t.shape != shape or (shape[2] > 1 and t.stride(2) != 1):
            raise ValueError(f"{name} must be {shape} with unit stride on the vocabulary, got {tuple(t.shape)}")
    _refuse_i32(parents, "parents", (B, T))
    _refuse_i32(n_nodes, "n_nodes", (B,))
    if u.dtype != torch.float32 or not u.is_cuda:
        raise TypeError("u must be a cuda fp32 tensor")
    _refuse_devices(tokens, parents=parents, n_nodes=n_nodes, target_probs=target_probs, u=u, draft_probs=draft_probs)
    raise ValueError(f"u must be contiguous ({B},{T}), got {tuple(u.shape)}")


def verify_tree(tokens, parents, n_nodes, target_probs, u, draft_probs=None):
    """Walk each row's tree of drafted tokens; returns (path, n_path, next_token).

    tokens (B, T) int64, parents (B, T) int32 with parents[b, c] < c, n_nodes
    (B,) int32: node 0 is the last committed token, the others are drafts.
    target_probs (B, T, V) fp32: the target's distribution after each node;
    draft_probs (the same, or None): the distribution from which the children
    of each node were drawn independently. u (B, T) fp32 in [0, 1): u[b, c]
    decides on node c, u[b, 0] draws the next token. With draft_probs child c
    is accepted when u * q(x) < w(x), and a rejection leaves
    w = max(w - q, 0) / sum; without, children are taken with their probability
    under what the rejected ones left over. In both the accepted tokens and the
    next one are distributed as draws from the target. Sums are exact (64-bit
    integers in units of 2^-36), so the result is the same on every run.

    path (B, T) int32: accepted nodes, node 0 first, then -1; n_path (B,) int32;
    next_token (B,) int64, -1 where n_nodes is 0 or the row has no mass.
    """
    r = _native().verify_tree(tokens, parents, n_nodes, target_probs, u, draft_probs)
    if r is None:
        _refuse(tokens, parents, n_nodes, target_probs, u, draft_probs)
    if type(r) is int:
        _failed(r, "fxb_verify_tree")
    return r
