"""fxlm.paged: a paged KV cache and the attention that reads it.

The reference's sampler keeps no cache and re-runs the whole window for every
token (ml/fxlm/sample.py:63-73). Here the keys and values of committed tokens
live in pages of a pool, and one decoding step is
    tree_attention per layer   the nodes of a token tree (one node: plain
                               decoding) attend to the cache and to each other
                               and are written behind the sequence,
    verify_tree                (fxlm.speculate) picks the accepted path,
    kv_commit                  moves the path's keys and values together and
                               makes room for the next tree.
kv_fork shares, copies and frees the pages of whole sequences.

Layout: k and v (L, P, H, page, D), one pool for all layers; page_table (S, W)
int32, row s holding the page of each run of `page` tokens of sequence s, -1
behind n_pages[s]; lens (S,) int32; ref (P,) int32, the number of rows that
hold a page (0: free). All of it stays on the device, and every call can be
captured in a CUDA graph. A call that does not fit (no free page, an id outside
the pool) sets the device error word: `fxb200._lib.raise_on_device_error()`.

A decoding step makes these calls once a layer for a few microseconds of GPU
work, so the checks, the result and the launch are one native call
(csrc/bind.cpp); what is wrong with arguments that do not fit is looked for
here.
"""
import ctypes
import functools

import torch

from fxb200 import _lib, ops

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
MAX_NODES = 64


@functools.lru_cache(maxsize=None)
def _native():
    """The native wrappers, given the library's functions."""
    lib, module = _lib.load(), _lib.load_binding()
    names = ("fxb_tree_attn", "fxb_tree_attn_workspace", "fxb_tree_attn_workspace_zeroed", "fxb_verify_tree",
             "fxb_kv_commit", "fxb_kv_fork", "fxb_kv_fork_workspace")
    module.init(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names), ops.stream_workspace, "tree_attn")
    return module


def _failed(rc, what):
    """Raises for the library's error code: ValueError for arguments that it refuses before any launch."""
    if rc == _lib.FXB_EINVAL:
        raise ValueError(_lib.last_error())
    _lib.check(rc, what)


def _refuse_i32(t, name, shape):
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"{name} must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)}")


def _refuse_devices(first, **others):
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, other arguments on {first.device}")


def _refuse_table(t):
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"page_table must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError("page_table must be (rows, entries) with unit stride on the entries")


def tree_masks(parents):
    """(B, T) int64 masks of a tree given by `parents` (B, T; -1 for the root,
    parents[b, c] < c): bit j of mask[b, c] is set for c itself and its ancestors.
    A parent outside [0, c) counts as none, as in verify_tree."""
    B, T = parents.shape
    if T > MAX_NODES:
        raise ValueError(f"T={T}: at most {MAX_NODES} nodes")
    up = parents.long()
    mask = torch.ones((), dtype=torch.int64, device=parents.device) << torch.arange(T, device=parents.device)
    mask = mask.expand(B, T)
    up = torch.where(up < torch.arange(T, device=parents.device), up, -1)
    for _ in range(max(T - 1, 0).bit_length()):  # doubling: after k steps the 2^k nearest ancestors are in
        has = up >= 0
        at = up.clamp(min=0)
        mask, up = mask | torch.where(has, mask.gather(1, at), 0), torch.where(has, up.gather(1, at), -1)
    return mask.contiguous()


def _refuse_tree(q, k, v, kp, vp, page_table, ctx_lens, n_nodes, tree_mask, out):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or kp.dim() != 4 or vp.dim() != 4:
        raise ValueError("q, k, v must be (B,T,H,D) and the pages (P,H,page,D)")
    dt = q.dtype
    if dt not in _DTYPES or not (k.dtype == v.dtype == kp.dtype == vp.dtype == dt):
        raise TypeError(f"q, k, v and the pages must share bf16, fp16 or fp32 ({dt}, {k.dtype}, {v.dtype}, "
                        f"{kp.dtype}, {vp.dtype})")
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} not supported (64 or 128)")
    if T > MAX_NODES:
        raise ValueError(f"T={T}: at most {MAX_NODES} nodes")
    if tuple(k.shape) != (B, T, Hkv, D) or v.shape != k.shape or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"shape mismatch: q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if tuple(kp.shape) != (kp.shape[0], Hkv, kp.shape[2], D) or vp.shape != kp.shape:
        raise ValueError(f"pages must share (P,{Hkv},page,{D}): {tuple(kp.shape)} {tuple(vp.shape)}")
    if not (q.is_cuda and k.is_cuda and v.is_cuda and kp.is_cuda and vp.is_cuda):
        raise TypeError("q, k, v and the pages must be cuda tensors")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, kp, vp)):
        raise ValueError("tree_attention has no backward pass: call it under torch.no_grad(), or with tensors that "
                         "require no gradient")
    _refuse_table(page_table)
    if page_table.shape[0] != B:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for a batch of {B}")
    if tree_mask.dtype != torch.int64 or not tree_mask.is_cuda:
        raise TypeError("tree_mask must be a cuda int64 tensor")
    if tuple(tree_mask.shape) != (B, T) or (T > 1 and tree_mask.stride(1) != 1):
        raise ValueError(f"tree_mask must be ({B},{T}) with unit stride on the nodes")
    if out is not None and (tuple(out.shape) != (B, T, Hq, D) or out.dtype != dt or not out.is_cuda):
        raise ValueError(f"out must be {(B, T, Hq, D)} {dt} on the GPU")
    _refuse_i32(ctx_lens, "ctx_lens", (B,))
    _refuse_i32(n_nodes, "n_nodes", (B,))
    _refuse_devices(q, k=k, v=v, k_pages=kp, v_pages=vp, page_table=page_table, ctx_lens=ctx_lens, n_nodes=n_nodes,
                    tree_mask=tree_mask, out=out)
    raise ValueError("the last axis of every tensor must be contiguous")


def tree_attention(q, k, v, k_pages, v_pages, page_table, ctx_lens, n_nodes, tree_mask, scale=None,
                   out=None):
    """Attention of tree nodes over a paged cache; returns o (B, T, Hq, D).

    q (B, T, Hq, D); k, v (B, T, Hkv, D) of the nodes, Hq a multiple of Hkv;
    k_pages, v_pages (P, Hkv, page, D) of one layer: views with unit stride on
    D (slices of a fused projection need no copy). Node t of row b sees the
    cache slots [0, ctx_lens[b]) and the nodes j < n_nodes[b] whose bit is set
    in tree_mask[b, t] (int64; one tree for all rows: tree_mask.expand(B, T)).
    k and v of the nodes j < n_nodes[b] are written to the slots
    ctx_lens[b] + j, which the row has to hold (kv_reserve or kv_commit's room).
    Rows t >= n_nodes[b], and rows that see nothing, are zeros. T <= 64, D 64 or 128, bf16 / fp16 / fp32; scale (1 / sqrt(D) by
    default) positive. There is no backward pass: tensors that require a
    gradient are refused while gradients are enabled.
    """
    o = _native().tree_attention(q, k, v, k_pages, v_pages, page_table, ctx_lens, n_nodes, tree_mask, scale, out)
    if o is None:
        _refuse_tree(q, k, v, k_pages, v_pages, page_table, ctx_lens, n_nodes, tree_mask, out)
    if type(o) is int:
        _failed(o, "fxb_tree_attn")
    return o


def _refuse_cache(k, v, page_table, n_pages, lens, ref):
    """Raises if something is wrong with a cache (k None: its table alone); returns its number of rows."""
    _refuse_table(page_table)
    S = page_table.shape[0]
    if ref.dim() != 1:
        raise ValueError(f"ref must be (P,), got {tuple(ref.shape)}")
    P = ref.shape[0]
    for t, name, n in ((n_pages, "n_pages", S), (lens, "lens", S), (ref, "ref", P)):
        _refuse_i32(t, name, (n,))
    _refuse_devices(page_table, n_pages=n_pages, lens=lens, ref=ref, k=k, v=v)
    if k is None:
        return S
    if k.dim() != 5 or v.shape != k.shape or k.shape[1] != P:
        raise ValueError(f"k and v must share (L,{P},H,page,D): {tuple(k.shape)} {tuple(v.shape)}")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError(f"k and v must share bf16, fp16 or fp32 ({k.dtype}, {v.dtype})")
    if not (k.is_cuda and v.is_cuda):
        raise TypeError("k and v must be cuda tensors")
    if k.stride(4) != 1 or v.stride(4) != 1:
        raise ValueError("the last axis of k and v must be contiguous")
    return S


def _refuse_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room, out):
    S = _refuse_cache(k, v, page_table, n_pages, lens, ref)
    if path is not None:
        if path.dim() != 2:
            raise ValueError(f"path must be ({S}, T), got {tuple(path.shape)}")
        if not 1 <= path.shape[1] <= MAX_NODES:
            raise ValueError(f"path of T={path.shape[1]} tokens: 1 to {MAX_NODES}")
        _refuse_i32(path, "path", (S, path.shape[1]))
        _refuse_i32(n_path, "n_path", (S,))
    for t, name in ((room, "room"), (out, "out")):
        if t is not None:
            _refuse_i32(t, name, (S,))
    _refuse_devices(page_table, path=path, n_path=n_path, room=room, out=out)
    raise ValueError("sizes of 2^31 and more")


def kv_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room=None, out=None):
    """Commit `path` of every row; returns the new lengths (S,) int32.

    Token i < n_path[s] moves from slot lens[s] + path[s, i] to lens[s] + i in
    every layer (path (S, T) int32 ascends strictly, as verify_tree returns it),
    the returned lengths are lens + n_path, and rows with room[s] > 0 are given
    pages for that many slots behind the new length: the lowest-numbered free
    ones, rows in order, none at all if the pool does not have enough.
    page_table, n_pages and ref are updated in place, lens is not; `out`, where
    given, receives the lengths and is none of the other arguments.
    """
    r = _native().kv_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room, out, 0)
    if r is None:
        _refuse_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room, out)
    if type(r) is int:
        _failed(r, "fxb_kv_commit")
    return r


def kv_reserve(page_table, n_pages, lens, ref, room, page):
    """Give every row pages for room[s] (S,) int32 slots behind lens[s], the
    lowest-numbered free ones, rows in order (kv_commit without a path)."""
    r = _native().kv_commit(None, None, page_table, n_pages, lens, ref, None, None, room, None, page)
    if r is None:
        _refuse_commit(None, None, page_table, n_pages, lens, ref, None, None, room, None)
    if type(r) is int:
        _failed(r, "fxb_kv_commit")


def kv_fork(k, v, page_table, n_pages, lens, ref, parents):
    """Row s becomes a fork of row parents[s] (S,) int32 as it was before the
    call; parents[s] == s keeps it, -1 empties it. Full pages are shared; a last
    page that is only partly filled stays with one row and is copied, in every
    layer, for the others. Updates all arrays in place; nothing changes if the
    pool lacks pages or a parent is out of range."""
    r = _native().kv_fork(k, v, page_table, n_pages, lens, ref, parents)
    if r is None:
        _refuse_i32(parents, "parents", (_refuse_cache(k, v, page_table, n_pages, lens, ref),))
        _refuse_devices(page_table, parents=parents)
        raise ValueError("sizes of 2^31 and more")
    if type(r) is int:
        _failed(r, "fxb_kv_fork")
