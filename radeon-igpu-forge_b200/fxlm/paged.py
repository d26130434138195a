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
"""
import ctypes
import math

import torch

from fxb200 import _lib, ops

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
MAX_NODES = 64


def _i32(t, name, shape):
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"{name} must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)}")
    return t.data_ptr()


def _table(t, name="page_table"):
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"{name} must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be (rows, entries) with unit stride on the entries")
    return t.shape


def tree_masks(parents):
    """(B, T) int64 masks of a tree given by `parents` (B, T; -1 for the root,
    parents[b, c] < c): bit j of mask[b, c] is set for c itself and its ancestors."""
    B, T = parents.shape
    if T > MAX_NODES:
        raise ValueError(f"T={T}: at most {MAX_NODES} nodes")
    par = parents.long()
    mask = torch.zeros(B, T, dtype=torch.int64, device=parents.device)
    for c in range(T):
        up = mask.gather(1, par[:, c:c + 1].clamp(min=0))[:, 0] if c else 0
        own = 1 << c if c < 63 else -(1 << 63)
        mask[:, c] = torch.where(par[:, c] >= 0, up, 0) | own
    return mask


def tree_attention(q, k, v, k_pages, v_pages, page_table, ctx_lens, n_nodes, tree_mask, scale=None,
                   out=None):
    """Attention of tree nodes over a paged cache; returns o (B, T, Hq, D).

    q (B, T, Hq, D); k, v (B, T, Hkv, D) of the nodes, Hq a multiple of Hkv;
    k_pages, v_pages (P, Hkv, page, D) of one layer: views with unit stride on
    D (slices of a fused projection need no copy). Node t of row b sees the
    cache slots [0, ctx_lens[b]) and the nodes j < n_nodes[b] whose bit is set
    in tree_mask[b, t] (int64). k and v of the nodes j < n_nodes[b] are written
    to the slots ctx_lens[b] + j, which the row has to hold (kv_reserve or
    kv_commit's room). Rows t >= n_nodes[b], and rows that see nothing, are
    zeros. T <= 64, D 64 or 128, bf16 / fp16 / fp32.
    """
    if q.dim() != 4 or k.dim() != 4 or k_pages.dim() != 4:
        raise ValueError("q, k, v must be (B,T,H,D) and the pages (P,H,page,D)")
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    P, _, page, _ = k_pages.shape
    dt = q.dtype
    if dt not in _DTYPES or not (k.dtype == v.dtype == k_pages.dtype == v_pages.dtype == dt):
        raise TypeError(f"q, k, v and the pages must share bf16, fp16 or fp32 ({dt}, {k.dtype}, {v.dtype}, "
                        f"{k_pages.dtype}, {v_pages.dtype})")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} not supported (64 or 128)")
    if T > MAX_NODES:
        raise ValueError(f"T={T}: at most {MAX_NODES} nodes")
    if tuple(k.shape) != (B, T, Hkv, D) or v.shape != k.shape or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"shape mismatch: q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if tuple(k_pages.shape) != (P, Hkv, page, D) or v_pages.shape != k_pages.shape:
        raise ValueError(f"pages must share (P,{Hkv},page,{D}): {tuple(k_pages.shape)} {tuple(v_pages.shape)}")
    if not (q.is_cuda and k.is_cuda and v.is_cuda and k_pages.is_cuda and v_pages.is_cuda):
        raise TypeError("q, k, v and the pages must be cuda tensors")
    rows, W = _table(page_table)
    if rows != B:
        raise ValueError(f"page_table has {rows} rows for a batch of {B}")
    lens, n = _i32(ctx_lens, "ctx_lens", (B,)), _i32(n_nodes, "n_nodes", (B,))
    if tree_mask.dtype != torch.int64 or not tree_mask.is_cuda:
        raise TypeError("tree_mask must be a cuda int64 tensor")
    if tuple(tree_mask.shape) != (B, T) or (T > 1 and tree_mask.stride(1) != 1):
        raise ValueError(f"tree_mask must be ({B},{T}) with unit stride on the nodes")
    if out is None:
        out = torch.empty((B, T, Hq, D), device=q.device, dtype=dt)
    elif tuple(out.shape) != (B, T, Hq, D) or out.dtype != dt or not out.is_cuda:
        raise ValueError(f"out must be {(B, T, Hq, D)} {dt} on the GPU")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    sq, sk, sv, so, skp, svp = (q.stride(), k.stride(), v.stride(), out.stride(), k_pages.stride(),
                                v_pages.stride())
    if not sq[3] == sk[3] == sv[3] == so[3] == skp[3] == svp[3] == 1:
        raise ValueError("the last axis of every tensor must be contiguous")
    if B == 0 or T == 0:
        return out
    lib = _lib.load()
    code = _lib.DTYPE_CODE[dt]
    shape = (code, B, T, Hq, Hkv, D)
    nbytes = lib.fxb_tree_attn_workspace(*shape)
    ws = ops.stream_workspace("tree_attn", q.device, nbytes, lib.fxb_tree_attn_workspace_zeroed(*shape))
    a = _lib.TreeAttnArgs(
        code, B, T, Hq, Hkv, D, page, P, W, scale,
        q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(), sk[0], sk[1], sk[2],
        v.data_ptr(), sv[0], sv[1], sv[2], out.data_ptr(), so[0], so[1], so[2],
        k_pages.data_ptr(), skp[0], skp[1], skp[2], v_pages.data_ptr(), svp[0], svp[1], svp[2],
        page_table.data_ptr(), max(page_table.stride(0), W), lens, n,
        tree_mask.data_ptr(), max(tree_mask.stride(0), T), ws.data_ptr(), nbytes)
    _lib.check(lib.fxb_tree_attn(ctypes.byref(a), _lib.stream_ptr(q.device)), "fxb_tree_attn")
    return out


def _kv_args(k, v, page_table, n_pages, lens, ref):
    S, W = _table(page_table)
    if ref.dim() != 1:
        raise ValueError(f"ref must be (P,), got {tuple(ref.shape)}")
    P = ref.shape[0]
    np_, ln, rf = _i32(n_pages, "n_pages", (S,)), _i32(lens, "lens", (S,)), _i32(ref, "ref", (P,))
    tail = (S, W, page_table.data_ptr(), max(page_table.stride(0), W), np_, ln, rf)
    if k is None:
        return (0, 0, P, 0), (None, 0, 0, 0, 0, None, 0, 0, 0, 0) + tail
    if k.dim() != 5 or v.shape != k.shape or k.shape[1] != P:
        raise ValueError(f"k and v must share (L,{P},H,page,D): {tuple(k.shape)} {tuple(v.shape)}")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError(f"k and v must share bf16, fp16 or fp32 ({k.dtype}, {v.dtype})")
    if not (k.is_cuda and v.is_cuda):
        raise TypeError("k and v must be cuda tensors")
    sk, sv = k.stride(), v.stride()
    if sk[4] != 1 or sv[4] != 1:
        raise ValueError("the last axis of k and v must be contiguous")
    return ((k.element_size(), k.shape[0], P, k.shape[2]),
            (k.data_ptr(), sk[0], sk[1], sk[2], sk[3], v.data_ptr(), sv[0], sv[1], sv[2], sv[3]) + tail)


def kv_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room=None, out=None):
    """Commit `path` of every row; returns the new lengths (S,) int32.

    Token i < n_path[s] moves from slot lens[s] + path[s, i] to lens[s] + i in
    every layer (path (S, T) int32 ascends strictly, as verify_tree returns it),
    the returned lengths are lens + n_path, and rows with room[s] > 0 are given
    pages for that many slots behind the new length: the lowest-numbered free
    ones, rows in order, none at all if the pool does not have enough.
    page_table, n_pages and ref are updated in place, lens is not.
    """
    head, rest = _kv_args(k, v, page_table, n_pages, lens, ref)
    S = page_table.shape[0]
    if path.dim() != 2:
        raise ValueError(f"path must be ({S}, T), got {tuple(path.shape)}")
    T = path.shape[1]
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"path of T={T} tokens: 1 to {MAX_NODES}")
    pp, pn = _i32(path, "path", (S, T)), _i32(n_path, "n_path", (S,))
    pr = _i32(room, "room", (S,)) if room is not None else None
    out = torch.empty_like(lens) if out is None else out
    po = _i32(out, "out", (S,))
    if S == 0:
        return out
    a = _lib.KvArgs(*head, k.shape[3], k.shape[4], *rest)
    _lib.check(_lib.load().fxb_kv_commit(ctypes.byref(a), pp, T, T, pn, pr, po, _lib.stream_ptr(lens.device)),
               "fxb_kv_commit")
    return out


def kv_reserve(page_table, n_pages, lens, ref, room, page):
    """Give every row pages for room[s] (S,) int32 slots behind lens[s], the
    lowest-numbered free ones, rows in order (kv_commit without a path)."""
    head, rest = _kv_args(None, None, page_table, n_pages, lens, ref)
    S = page_table.shape[0]
    pr = _i32(room, "room", (S,))
    if S == 0:
        return
    same = torch.empty_like(lens)
    a = _lib.KvArgs(*head, page, 0, *rest)
    _lib.check(_lib.load().fxb_kv_commit(ctypes.byref(a), None, 0, 0, None, pr, same.data_ptr(),
                                         _lib.stream_ptr(lens.device)), "fxb_kv_commit")


def kv_fork(k, v, page_table, n_pages, lens, ref, parents):
    """Row s becomes a fork of row parents[s] (S,) int32 as it was before the
    call; parents[s] == s keeps it, -1 empties it. Full pages are shared; a last
    page that is only partly filled stays with one row and is copied, in every
    layer, for the others. Updates all arrays in place; nothing changes if the
    pool lacks pages or a parent is out of range."""
    head, rest = _kv_args(k, v, page_table, n_pages, lens, ref)
    S, W = page_table.shape
    pp = _i32(parents, "parents", (S,))
    if S == 0:
        return
    lib = _lib.load()
    ws = torch.empty(lib.fxb_kv_fork_workspace(S, W), device=lens.device, dtype=torch.uint8)
    a = _lib.KvArgs(*head, k.shape[3], k.shape[4], *rest)
    _lib.check(lib.fxb_kv_fork(ctypes.byref(a), pp, ws.data_ptr(), _lib.stream_ptr(lens.device)), "fxb_kv_fork")
