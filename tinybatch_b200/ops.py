"""Thin torch-tensor wrappers over the C ABI (one function per fused kernel).

Every function checks shapes on the host, calls the library on the current
CUDA stream and raises ``NativeError`` on a nonzero return code.  Scratch
buffers come from a ``Scratch`` arena owned by the caller (nothing here
allocates per call except when no arena is given).
"""
from __future__ import annotations

import ctypes
from array import array

import torch

from . import _native as N
from ._native import ptr


class Scratch:
    """A zero-initialised device arena reused by every call that needs
    split-K or split-KV scratch.  Grows (re-zeroed) when a call needs more."""

    def __init__(self, device, nbytes: int = 0):
        self.device = torch.device(device)
        self.buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=self.device)
        self.version = 0        # bumped on every growth (captured graphs must check it)
        self._retired: list[torch.Tensor] = []

    def get(self, nbytes: int) -> tuple[int | None, int]:
        if nbytes == 0:
            return None, 0
        if nbytes > self.buf.numel():
            # the old buffer stays alive: a graph captured on it never reads freed memory
            self._retired.append(self.buf)
            self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
            self.version += 1
        return self.buf.data_ptr(), self.buf.numel()


def _gemm_scratch(scratch: Scratch | None, device, M, n_cols, bn, splits, split_mode):
    """Scratch for a GEMM call: none for cluster split-K (the default),
    caller scratch for ``split_mode="global"``."""
    if splits <= 1 or split_mode == "cluster":
        return None, 0, None
    if split_mode != "global":
        raise ValueError(f"split_mode must be 'cluster' or 'global', not {split_mode!r}")
    return _scratch(scratch, device, N.load().tb_gemm_scratch_bytes(M, n_cols, bn, splits))


def _scratch(scratch: Scratch | None, device, nbytes: int):
    if nbytes == 0:
        return None, 0, None
    if scratch is None:
        scratch = Scratch(device, nbytes)
    p, n = scratch.get(nbytes)
    return p, n, scratch


def _sq(sq):
    """(ptr, parts, ld) of a deferred-norm partial-sum buffer [parts, ld] or None."""
    if sq is None:
        return None, 0, 0
    return ptr(sq), sq.shape[0], sq.stride(0)


def linear(x, w, out, *, sq=None, inv_d=0.0, eps=0.0, bn=128, splits=1, scratch=None,
           split_mode="cluster"):
    lib = N.load()
    M, K = x.shape
    Nn = w.shape[0]
    ws, wsn, _ = _gemm_scratch(scratch, x.device, M, Nn, bn, splits, split_mode)
    sp, parts, sld = _sq(sq)
    N.check(lib.tb_linear(ptr(x), x.stride(0), ptr(w), w.stride(0), M, Nn, K, sp, parts, sld,
                          inv_d, eps, ptr(out), out.stride(0), int(out.dtype == torch.float32),
                          bn, splits, ws, wsn, N.stream_ptr()), "tb_linear")
    return out


def qkv_rope_kv(x, w_qkv, bias, *, n_q_heads, n_kv_heads, head_dim, sq, inv_d, eps,
                rope_cos, rope_sin, positions, slots, q_out, kv_pool, block_size,
                bn=128, splits=1, scratch=None, split_mode="cluster"):
    lib = N.load()
    M, K = x.shape
    Nn = w_qkv.shape[0]
    ws, wsn, _ = _gemm_scratch(scratch, x.device, M, Nn, bn, splits, split_mode)
    sp, parts, sld = _sq(sq)
    N.check(lib.tb_qkv_rope_kv(ptr(x), x.stride(0), ptr(w_qkv), w_qkv.stride(0), ptr(bias), M,
                               K, n_q_heads, n_kv_heads, head_dim, sp, parts, sld, inv_d, eps,
                               ptr(rope_cos), ptr(rope_sin), rope_cos.shape[0], ptr(positions),
                               ptr(slots), ptr(q_out), q_out.stride(0), ptr(kv_pool),
                               block_size, bn, splits, ws, wsn, N.stream_ptr()),
            "tb_qkv_rope_kv")


def gate_up_swiglu(x, w_gu, act, *, n_feat, sq, inv_d, eps, bn=128, splits=1, scratch=None,
                   split_mode="cluster"):
    lib = N.load()
    M, K = x.shape
    Nn = w_gu.shape[0]
    ws, wsn, _ = _gemm_scratch(scratch, x.device, M, Nn, bn, splits, split_mode)
    sp, parts, sld = _sq(sq)
    N.check(lib.tb_gate_up_swiglu(ptr(x), x.stride(0), ptr(w_gu), w_gu.stride(0), M, K, n_feat,
                                  sp, parts, sld, inv_d, eps, ptr(act), act.stride(0), bn,
                                  splits, ws, wsn, N.stream_ptr()),
            "tb_gate_up_swiglu")
    return act


def row_parts(n_cols: int, bn: int, splits: int, split_mode: str = "cluster") -> int:
    """Rows of deferred-norm partial sums a row-parallel call writes: one per
    column tile, or per (column tile, cluster member) with cluster split-K."""
    tiles = -(-n_cols // bn)
    return tiles * splits if (splits > 1 and split_mode == "cluster") else tiles


def row_linear_residual(x, w, h, g_next, hg, sq_out, *, row_dst=None, hg2=None, sq2=None,
                        bn=128, splits=1, scratch=None, split_mode="cluster"):
    lib = N.load()
    M, K = x.shape
    Nn = w.shape[0]
    ws, wsn, _ = _gemm_scratch(scratch, x.device, M, Nn, bn, splits, split_mode)
    N.check(lib.tb_row_linear_residual(
        ptr(x), x.stride(0), ptr(w), w.stride(0), M, Nn, K, ptr(h), h.stride(0), ptr(g_next),
        ptr(hg), hg.stride(0), ptr(sq_out), sq_out.stride(0), ptr(row_dst), ptr(hg2),
        ptr(sq2), sq2.stride(0) if sq2 is not None else 0, bn, splits, ws, wsn,
        N.stream_ptr()), "tb_row_linear_residual")


def paged_attention_decode(q, out, kv_pool, *, n_q_heads, n_kv_heads, head_dim, block_size,
                           block_tables, q_start, q_len, ctx_len, max_ctx, split_tokens=512,
                           seq_order=None, scratch=None):
    """``seq_order`` (optional int32 [n]): the order in which sequences are
    dispatched (e.g. longest first)."""
    lib = N.load()
    n = ctx_len.shape[0]
    ws, wsn, _ = _scratch(scratch, q.device, lib.tb_attention_scratch_bytes(
        n, n_kv_heads, head_dim, max_ctx, split_tokens))
    N.check(lib.tb_paged_attention_decode(
        ptr(q), q.stride(0), ptr(out), out.stride(0), ptr(kv_pool), kv_pool.shape[0],
        n_q_heads, n_kv_heads, head_dim, block_size, ptr(block_tables), block_tables.stride(0),
        ptr(q_start), ptr(q_len), ptr(ctx_len), ptr(seq_order), n, max_ctx, split_tokens, ws,
        wsn, N.stream_ptr()), "tb_paged_attention_decode")


def paged_attention_prefill(q, out, kv_pool, *, n_q_heads, n_kv_heads, head_dim, block_size,
                            block_tables, q_start, q_len, ctx_len, work):
    if work.dim() != 2 or work.shape[1] != 2 or work.dtype != torch.int32:
        raise ValueError("work must be an int32 [n_work, 2] tensor of (sequence, row tile)")
    lib = N.load()
    n = ctx_len.shape[0]
    N.check(lib.tb_paged_attention_prefill(
        ptr(q), q.stride(0), ptr(out), out.stride(0), ptr(kv_pool), kv_pool.shape[0],
        n_q_heads, n_kv_heads, head_dim, block_size, ptr(block_tables), block_tables.stride(0),
        ptr(q_start), ptr(q_len), ptr(ctx_len), n, ptr(work), work.shape[0], N.stream_ptr()),
        "tb_paged_attention_prefill")


# ------------------------------------------------- speculative decoding
#
# These calls check types, shapes, devices and strides of every tensor (a
# mistake raises ValueError before anything is launched) and run on the
# tensors' own device, on its current stream.

def _device(t: torch.Tensor) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError("expected CUDA tensors")
    return dev


# One function per kind of argument, a single condition each: a decode step's
# calls are a few microseconds of GPU work, so the host's share counts.

def _refuse(name: str, t: torch.Tensor, want: str, dev: int):
    raise ValueError(f"{name}: expected {want} on cuda:{dev}, got {tuple(t.shape)} {t.dtype} on "
                     f"{t.device}, strides {t.stride()}")


def _vec(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, dev: int) -> int:
    """Data pointer of a contiguous argument of exactly this shape."""
    if (t.dtype is dtype and t.shape == shape and t.get_device() == dev
            and t.is_contiguous()):
        return t.data_ptr()
    _refuse(name, t, f"a contiguous {shape} {dtype} tensor", dev)


def _mat(name: str, t: torch.Tensor, dtype: torch.dtype, rows: int | None, dev: int):
    """(pointer, row pitch, columns) of a 2-d argument with contiguous rows; the C
    entries take 32-bit pitches."""
    shape = t.shape
    if t.dtype is dtype and len(shape) == 2 and t.get_device() == dev:
        n, cols = shape
        pitch, step = t.stride()
        if (rows is None or n == rows) and (step == 1 or cols <= 1) and (
                pitch < 0x80000000 or n <= 1):
            return t.data_ptr(), (pitch if n > 1 else cols), cols
    _refuse(name, t, f"a 2-d {dtype} tensor of {'any' if rows is None else rows} contiguous rows",
            dev)


# torch.cuda.current_stream / current_device without their objects and checks
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_I32, _I64, _F32, _BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16


def _run_on(dev: int, what: str, fn, *args) -> None:
    """Call ``fn(*args, stream)`` on device ``dev``'s current stream."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        N.check(rc, what)


def paged_attention_tree(q, out, kv_pool, *, n_q_heads, n_kv_heads, head_dim, block_size,
                         block_tables, q_start, q_len, ctx_len, tree_mask, max_q=None,
                         max_ctx=0, ctx_total=0):
    """Attention of drafted tokens over the paged cache: row ``q_start[s] + i``
    is node i of sequence s's draft tree, its K/V at position ``ctx_len[s] -
    q_len[s] + i``; it sees every earlier position and the nodes whose bits
    are set in its row of ``tree_mask`` (int64 ``[rows, words]``, bit ``j %
    64`` of word ``j // 64``; ``runtime.tree_masks`` builds it).  Rows that
    see nothing get zeros, rows of no sequence are left as they were.

    ``max_q``: the largest ``q_len`` (default: as many as the mask can name); a
    sequence that has more sets the status word and its rows are not written.
    ``max_ctx`` / ``ctx_total``: the longest context and their sum where the
    caller knows them (they only choose how a context is shared out)."""
    lib = N.load()
    dev = _device(q)
    rows, n = len(q), len(ctx_len)
    qp, ldq, cols = _mat("q", q, _BF16, rows, dev)
    op, ldo, ocols = _mat("out", out, _BF16, rows, dev)
    if cols != n_q_heads * head_dim or ocols != cols:
        raise ValueError(f"q and out: expected {n_q_heads * head_dim} columns, got {cols} and {ocols}")
    blocks = len(kv_pool)
    pp = _vec("kv_pool", kv_pool, _BF16, (blocks, 2, n_kv_heads, block_size, head_dim), dev)
    bp, ldb, width = _mat("block_tables", block_tables, _I32, n, dev)
    mp, ldm, words = _mat("tree_mask", tree_mask, _I64, rows, dev)
    seqs = (n,)
    _run_on(dev, "tb_paged_attention_tree", lib.tb_paged_attention_tree, qp, ldq, op, ldo, rows, pp,
            blocks, n_q_heads, n_kv_heads, head_dim, block_size, bp, ldb, width,
            _vec("q_start", q_start, _I32, seqs, dev), _vec("q_len", q_len, _I32, seqs, dev),
            _vec("ctx_len", ctx_len, _I32, seqs, dev), n, mp, ldm, words,
            min(rows, 64 * words) if max_q is None else max_q or 1, max_ctx, ctx_total)


def _tree(ids, parents, q_start, q_len, n_accepted, path, next_ids, dev):
    """Sizes and pointers of the arguments both verifications share."""
    rows, seqs = ids.shape, q_len.shape
    if len(rows) != 1 or len(seqs) != 1:
        raise ValueError("ids and q_len: expected 1-d tensors")
    return (rows, seqs[0],
            (_vec("ids", ids, _I32, rows, dev), _vec("parents", parents, _I32, rows, dev),
             _vec("q_start", q_start, _I32, seqs, dev), _vec("q_len", q_len, _I32, seqs, dev)),
            (_vec("n_accepted", n_accepted, _I32, seqs, dev),
             *_mat("path", path, _I32, seqs[0], dev), _vec("next_ids", next_ids, _I32, seqs, dev)))


def verify_drafts_greedy(ids, parents, q_start, q_len, target_ids, n_accepted, path, next_ids, *,
                         max_q=0):
    """Walk every sequence's draft tree along the target's choices: from the
    root to the first child whose id is ``target_ids`` at its parent's row, as
    long as there is one.  Writes the accepted nodes (root first, then -1) to
    ``path`` ``[n, width]``, how many drafts they are to ``n_accepted`` and
    the target's choice after the last of them to ``next_ids``."""
    lib = N.load()
    dev = _device(ids)
    rows, n, tree, outs = _tree(ids, parents, q_start, q_len, n_accepted, path, next_ids, dev)
    tp = _vec("target_ids", target_ids, _I32, rows, dev)
    _run_on(dev, "tb_verify_drafts_greedy", lib.tb_verify_drafts_greedy, *tree, n, rows[0], max_q,
            tp, *outs)


def verify_drafts(ids, parents, q_start, q_len, probs, uniforms, n_accepted, path, next_ids, *,
                  draft_probs=None, draft_rows=None, max_q=0):
    """Verify draft trees by speculative sampling, so that the accepted tokens
    and ``next_ids`` follow the target's distribution.

    ``probs`` ``[rows, vocab]`` fp32: the target's distribution after each
    node.  ``draft_probs`` ``[k, vocab]`` fp32 with ``draft_rows`` ``[rows]``
    int32: the distribution each node's children were drawn from without
    replacement (-1, or both None: picked outright).  ``uniforms`` ``[rows]``
    fp32 in [0, 1): one for each draft's test, the root's for the final
    sample.  Outputs as ``verify_drafts_greedy``."""
    lib = N.load()
    dev = _device(ids)
    rows, n, tree, outs = _tree(ids, parents, q_start, q_len, n_accepted, path, next_ids, dev)
    pp, ldp, vocab = _mat("probs", probs, _F32, rows[0], dev)
    up = _vec("uniforms", uniforms, _F32, rows, dev)
    if (draft_probs is None) != (draft_rows is None):
        raise ValueError("draft_probs and draft_rows go together")
    draft = (None, 0, 0, None)
    if draft_probs is not None:
        dp, ldd, cols = _mat("draft_probs", draft_probs, _F32, None, dev)
        if cols != vocab:
            raise ValueError(f"draft_probs: expected {vocab} columns, got {cols}")
        # (without any distribution there is no address, and no row may name one)
        draft = (dp or pp, ldd, len(draft_probs), _vec("draft_rows", draft_rows, _I32, rows, dev))
    _run_on(dev, "tb_verify_drafts", lib.tb_verify_drafts, *tree, n, rows[0], max_q, pp, ldp, vocab,
            *draft, up, *outs)


class KVPools:
    """The layers' KV pools as one argument of the cache moves: checked once,
    their addresses in a host array.  Holds the tensors; a pool whose storage is
    exchanged needs a new one."""

    def __init__(self, pools):
        """``pools``: a list of ``[num_blocks, 2, n_kv, block_size, head_dim]``
        bf16 tensors, or one tensor with the layers stacked in front."""
        if isinstance(pools, torch.Tensor):
            shape, pitch = pools.shape, pools.stride()
            if len(shape) != 6 or shape[2] != 2:
                raise ValueError("stacked pools: expected [layers, num_blocks, 2, n_kv, block_size, "
                                 f"head_dim], got {tuple(shape)}")
            layers, blocks, _, heads, size, dim = shape
            token = size * dim
            if pools.dtype is not torch.bfloat16 or (
                    pitch[1:] != (2 * heads * token, heads * token, token, dim, 1)
                    and not (layers and pools[0].is_contiguous())):
                raise ValueError("pools must be bf16, each layer's contiguous")
            step = pitch[0] * 2
            if layers > 1 and step < blocks * heads * token * 4:
                raise ValueError("pools: layers overlap")
            first = pools.data_ptr()
            ptrs = range(first, first + layers * step, step) if layers > 1 else (first,) * layers
            self.device = _device(pools)
        else:
            pools = list(pools)
            shape = pools[0].shape if pools else ()
            if len(shape) != 5 or shape[1] != 2:
                raise ValueError("pools: expected tensors [num_blocks, 2, n_kv, block_size, head_dim], "
                                 f"got {tuple(shape)}")
            layers = len(pools)
            blocks, _, heads, size, dim = shape
            self.device = _device(pools[0])
            for t in pools:
                if (t.dtype is not torch.bfloat16 or t.shape != shape or not t.is_contiguous()
                        or t.get_device() != self.device):
                    raise ValueError("pools must be contiguous bf16 tensors of one shape and device")
            ptrs = [t.data_ptr() for t in pools]
            if len(set(ptrs)) != layers:
                raise ValueError("pools: a layer is listed twice")
        self.pools = pools
        self.addresses = array("Q", ptrs)      # what the first of args points to
        # the C calls' first arguments: the addresses, the layers, a pool's shape
        self.args = (self.addresses.buffer_info()[0], layers, blocks, heads, size, dim)


def _pools(pools) -> KVPools:
    return pools if isinstance(pools, KVPools) else KVPools(pools)


def keep_kv_path(pools, *, block_tables, q_len, ctx_len, path, n_accepted):
    """After a verification: in every layer, move the K/V of each sequence's
    accepted nodes (``path``, ``n_accepted`` as the verification wrote them)
    to the consecutive positions after the root.  ``pools``: ``KVPools``, or
    what it takes."""
    lib = N.load()
    kv = _pools(pools)
    dev = kv.device
    seqs = q_len.shape
    if len(seqs) != 1:
        raise ValueError("q_len: expected a 1-d tensor")
    _run_on(dev, "tb_keep_kv_path", lib.tb_keep_kv_path, *kv.args,
            *_mat("block_tables", block_tables, _I32, seqs[0], dev),
            _vec("q_len", q_len, _I32, seqs, dev), _vec("ctx_len", ctx_len, _I32, seqs, dev),
            *_mat("path", path, _I32, seqs[0], dev),
            _vec("n_accepted", n_accepted, _I32, seqs, dev), seqs[0])


def copy_kv_blocks(pools, pairs):
    """Copy block ``pairs[i, 0]`` to block ``pairs[i, 1]`` in every layer
    (``pairs`` int32 ``[n, 2]`` on the device).  No destination may be
    another pair's source or destination: such pairs are not made and set the
    status word.  ``pools``: ``KVPools``, or what it takes."""
    lib = N.load()
    kv = _pools(pools)
    n = len(pairs)
    _run_on(kv.device, "tb_copy_kv_blocks", lib.tb_copy_kv_blocks, *kv.args,
            _vec("pairs", pairs, _I32, (n, 2), kv.device), n)


def embed(ids, emb, g, h, hg, sq):
    lib = N.load()
    M = ids.shape[0]
    N.check(lib.tb_embed(ptr(ids), M, ptr(emb), emb.stride(0), emb.shape[1], emb.shape[0],
                         ptr(g), ptr(h), h.stride(0), ptr(hg), hg.stride(0), ptr(sq),
                         N.stream_ptr()), "tb_embed")


def argmax(logits, out):
    lib = N.load()
    M, V = logits.shape
    N.check(lib.tb_argmax(ptr(logits), logits.stride(0), M, V, ptr(out), N.stream_ptr()),
            "tb_argmax")
    return out


def max_active_clusters(bn: int, cluster: int) -> int:
    out = ctypes.c_int(0)
    N.check(N.load().tb_gemm_max_active_clusters(bn, cluster, ctypes.byref(out)),
            "tb_gemm_max_active_clusters")
    return out.value
