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
work, so the wrappers check everything in one expression and look for the
reason only when it fails; the C structs are packed in one call.
"""
import functools
import math
import struct

import torch

from fxb200 import _lib, ops

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_CODE = _lib.DTYPE_CODE
MAX_NODES = 64
_I32 = torch.int32

# fxb_tree_attn_args and fxb_kv_args (mirrored field by field in fxb200._lib)
_TREE_ARGS = struct.Struct("@9if32q")
_KV_ARGS = struct.Struct("@6i10q2i5q")


def _refuse_i32(t, name, shape):
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"{name} must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    raise ValueError(f"{name} must be contiguous {shape}, got {tuple(t.shape)}")


def _i32(t, name, shape):
    if not (t.dtype is _I32 and t.is_cuda and t.shape == shape and t.is_contiguous()):
        _refuse_i32(t, name, shape)
    return t.data_ptr()


def _table(t, name="page_table"):
    """(address, rows, entries, row stride) of a page table."""
    if t.dtype != torch.int32 or not t.is_cuda:
        raise TypeError(f"{name} must be a cuda int32 tensor, got {t.dtype} on {t.device}")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be (rows, entries) with unit stride on the entries")
    S, W = t.shape
    return t.data_ptr(), S, W, t.stride(0) if S > 1 else W


def tree_masks(parents):
    """(B, T) int64 masks of a tree given by `parents` (B, T; -1 for the root,
    parents[b, c] < c): bit j of mask[b, c] is set for c itself and its ancestors."""
    B, T = parents.shape
    if T > MAX_NODES:
        raise ValueError(f"T={T}: at most {MAX_NODES} nodes")
    up = parents.long()
    mask = torch.ones((), dtype=torch.int64, device=parents.device) << torch.arange(T, device=parents.device)
    mask = mask.expand(B, T)
    for _ in range(max(T - 1, 0).bit_length()):  # doubling: after k steps the 2^k nearest ancestors are in
        has = up >= 0
        at = up.clamp(min=0)
        mask, up = mask | torch.where(has, mask.gather(1, at), 0), torch.where(has, up.gather(1, at), -1)
    return mask.contiguous()


@functools.lru_cache(maxsize=1024)
def _tree_workspace(device, *shape):
    """(bytes, bytes that start at zero) for this device and shape."""
    lib = _lib.load()
    return lib.fxb_tree_attn_workspace(*shape), lib.fxb_tree_attn_workspace_zeroed(*shape)


def _refuse_tree(q, k, v, kp, vp, page_table, tree_mask, out):
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
    if _table(page_table)[1] != B:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for a batch of {B}")
    if tree_mask.dtype != torch.int64 or not tree_mask.is_cuda:
        raise TypeError("tree_mask must be a cuda int64 tensor")
    if tuple(tree_mask.shape) != (B, T) or (T > 1 and tree_mask.stride(1) != 1):
        raise ValueError(f"tree_mask must be ({B},{T}) with unit stride on the nodes")
    if out is not None and (tuple(out.shape) != (B, T, Hq, D) or out.dtype != dt or not out.is_cuda):
        raise ValueError(f"out must be {(B, T, Hq, D)} {dt} on the GPU")
    raise ValueError("the last axis of every tensor must be contiguous")


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
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or k_pages.dim() != 4 or v_pages.dim() != 4:
        raise ValueError("q, k, v must be (B,T,H,D) and the pages (P,H,page,D)")
    B, T, Hq, D = shape = q.shape
    Hkv = k.shape[2]
    P, _, page, _ = k_pages.shape
    dt = q.dtype
    q_sb, q_st, q_sh, q1 = q.stride()
    k_sb, k_st, k_sh, k1 = k.stride()
    v_sb, v_st, v_sh, v1 = v.stride()
    kp_sp, kp_sh, kp_st, kp1 = k_pages.stride()
    vp_sp, vp_sh, vp_st, vp1 = v_pages.stride()
    fits = (dt in _DTYPES and k.dtype == dt and v.dtype == dt and k_pages.dtype == dt and v_pages.dtype == dt
            and (D == 64 or D == 128) and T <= MAX_NODES and Hkv > 0 and Hq % Hkv == 0
            and k.shape == (B, T, Hkv, D) and v.shape == (B, T, Hkv, D)
            and k_pages.shape == (P, Hkv, page, D) and v_pages.shape == (P, Hkv, page, D)
            and q.is_cuda and k.is_cuda and v.is_cuda and k_pages.is_cuda and v_pages.is_cuda
            and page_table.dtype == torch.int32 and page_table.is_cuda and page_table.dim() == 2
            and page_table.shape[0] == B and page_table.stride(1) == 1 and tree_mask.dtype == torch.int64 and tree_mask.is_cuda
            and tree_mask.shape == (B, T) and (T == 1 or tree_mask.stride(1) == 1)
            and q1 == k1 == v1 == kp1 == vp1 == 1)
    if out is not None:
        fits = fits and out.shape == shape and out.dtype == dt and out.is_cuda and out.stride(3) == 1
    if not fits:
        _refuse_tree(q, k, v, k_pages, v_pages, page_table, tree_mask, out)
    lens, n = _i32(ctx_lens, "ctx_lens", (B,)), _i32(n_nodes, "n_nodes", (B,))
    if out is None:
        out = q.new_empty(shape)
    if B == 0 or T == 0:
        return out
    W, table_sb = page_table.shape[1], page_table.stride(0)
    o_sb, o_st, o_sh, _ = out.stride()
    code = _CODE[dt]
    device = q.get_device()
    stream = _lib.raw_stream(device)
    nbytes, zeroed = _tree_workspace(device, code, B, T, Hq, Hkv, D)
    ws = ops.stream_workspace("tree_attn", device, stream, nbytes, zeroed)
    args = _TREE_ARGS.pack(
        code, B, T, Hq, Hkv, D, page, P, W, 1.0 / math.sqrt(D) if scale is None else scale,
        q.data_ptr(), q_sb, q_st, q_sh, k.data_ptr(), k_sb, k_st, k_sh, v.data_ptr(), v_sb, v_st, v_sh,
        out.data_ptr(), o_sb, o_st, o_sh, k_pages.data_ptr(), kp_sp, kp_sh, kp_st,
        v_pages.data_ptr(), vp_sp, vp_sh, vp_st, page_table.data_ptr(), table_sb if B > 1 else W, lens, n,
        tree_mask.data_ptr(), tree_mask.stride(0) if B > 1 else T, ws.data_ptr(), nbytes)
    rc = _lib.load().fxb_tree_attn(args, stream)
    if rc:
        _lib.check(rc, "fxb_tree_attn")
    return out


def _kv_args(k, v, page_table, n_pages, lens, ref, page=0):
    """fxb_kv_args of a cache (k None: of its table alone) and its number of rows."""
    table, S, W, table_ss = _table(page_table)
    if ref.dim() != 1:
        raise ValueError(f"ref must be (P,), got {tuple(ref.shape)}")
    P = ref.shape[0]
    tail = (S, W, table, table_ss, _i32(n_pages, "n_pages", (S,)), _i32(lens, "lens", (S,)), _i32(ref, "ref", (P,)))
    if k is None:
        return _KV_ARGS.pack(0, 0, P, 0, page, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, *tail), S
    if k.dim() != 5 or v.shape != k.shape or k.shape[1] != P:
        raise ValueError(f"k and v must share (L,{P},H,page,D): {tuple(k.shape)} {tuple(v.shape)}")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError(f"k and v must share bf16, fp16 or fp32 ({k.dtype}, {v.dtype})")
    if not (k.is_cuda and v.is_cuda):
        raise TypeError("k and v must be cuda tensors")
    L, P, H, page, D = k.shape
    k_sl, k_sp, k_sh, k_st, k1 = k.stride()
    v_sl, v_sp, v_sh, v_st, v1 = v.stride()
    if k1 != 1 or v1 != 1:
        raise ValueError("the last axis of k and v must be contiguous")
    return _KV_ARGS.pack(k.element_size(), L, P, H, page, D, k.data_ptr(), k_sl, k_sp, k_sh, k_st,
                         v.data_ptr(), v_sl, v_sp, v_sh, v_st, *tail), S


def kv_commit(k, v, page_table, n_pages, lens, ref, path, n_path, room=None, out=None):
    """Commit `path` of every row; returns the new lengths (S,) int32.

    Token i < n_path[s] moves from slot lens[s] + path[s, i] to lens[s] + i in
    every layer (path (S, T) int32 ascends strictly, as verify_tree returns it),
    the returned lengths are lens + n_path, and rows with room[s] > 0 are given
    pages for that many slots behind the new length: the lowest-numbered free
    ones, rows in order, none at all if the pool does not have enough.
    page_table, n_pages and ref are updated in place, lens is not.
    """
    args, S = _kv_args(k, v, page_table, n_pages, lens, ref)
    if path.dim() != 2:
        raise ValueError(f"path must be ({S}, T), got {tuple(path.shape)}")
    T = path.shape[1]
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"path of T={T} tokens: 1 to {MAX_NODES}")
    pp, pn = _i32(path, "path", (S, T)), _i32(n_path, "n_path", (S,))
    pr = _i32(room, "room", (S,)) if room is not None else None
    if out is None:
        out = torch.empty_like(lens)
    po = _i32(out, "out", (S,))
    if S:
        rc = _lib.load().fxb_kv_commit(args, pp, T, T, pn, pr, po, _lib.raw_stream(lens.get_device()))
        if rc:
            _lib.check(rc, "fxb_kv_commit")
    return out


def kv_reserve(page_table, n_pages, lens, ref, room, page):
    """Give every row pages for room[s] (S,) int32 slots behind lens[s], the
    lowest-numbered free ones, rows in order (kv_commit without a path)."""
    args, S = _kv_args(None, None, page_table, n_pages, lens, ref, page)
    pr = _i32(room, "room", (S,))
    if S:
        same = torch.empty_like(lens)
        rc = _lib.load().fxb_kv_commit(args, None, 0, 0, None, pr, same.data_ptr(),
                                       _lib.raw_stream(lens.get_device()))
        if rc:
            _lib.check(rc, "fxb_kv_commit")


def kv_fork(k, v, page_table, n_pages, lens, ref, parents):
    """Row s becomes a fork of row parents[s] (S,) int32 as it was before the
    call; parents[s] == s keeps it, -1 empties it. Full pages are shared; a last
    page that is only partly filled stays with one row and is copied, in every
    layer, for the others. Updates all arrays in place; nothing changes if the
    pool lacks pages or a parent is out of range."""
    args, S = _kv_args(k, v, page_table, n_pages, lens, ref)
    pp = _i32(parents, "parents", (S,))
    if S:
        lib = _lib.load()
        ws = lens.new_empty((lib.fxb_kv_fork_workspace(S, page_table.shape[1]) + 3) // 4)
        rc = lib.fxb_kv_fork(args, pp, ws.data_ptr(), _lib.raw_stream(lens.get_device()))
        if rc:
            _lib.check(rc, "fxb_kv_fork")
