"""ctypes front-end of include/kv_cache.h: the 4-bit KV cache (RoPE and
quantising page write, rows read back, split decode attention) and the page
operators (fork, free and extend rows; compact a pool).

The 4-bit caches stand beside the bf16 pages of :mod:`time_b200.attn` and take
the same page tables; the page operators work on the pages of either, all
layers' K and V in one tensor ``[caches][pages][...]``.  A sequence of ``len``
tokens owns the first ``ceil(len / 16)`` entries of its page-table row and a
page in no row is free, so a request is freed by leaving its row out of the
next fork.
"""
from __future__ import annotations

import functools
from ctypes import c_float, c_int, c_size_t, c_void_p

from . import attn as A
from . import moe as M

HEAD_DIM, PAGE, GROUP = A.HEAD_DIM, A.PAGE, 32
CODE_BYTES = PAGE * HEAD_DIM // 2
PAGE4_BYTES = CODE_BYTES + PAGE * (HEAD_DIM // GROUP) * 2      # one page of one kv head

_lib = None


def lib():
    global _lib
    if _lib is None:
        k = M.libs()["libkernels.so"]
        k.attn_kv4_page_bytes.argtypes = [c_int]
        k.attn_kv4_page_bytes.restype = c_size_t
        k.attn_kv4_rope_write_rows.argtypes = [c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                                               c_void_p, c_int, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p,
                                               c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]
        k.attn_kv4_read_rows.argtypes = [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int,
                                         c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p]
        k.attn_kv4_split_tokens.argtypes = [c_int, c_int, c_int]
        k.attn_kv4_decode_workspace_bytes.argtypes = [c_int, c_int, c_int]
        k.attn_kv4_decode_workspace_bytes.restype = c_size_t
        k.attn_kv4_decode_rows.argtypes = [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_void_p, c_int,
                                           c_void_p, c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int,
                                           c_void_p, c_size_t, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p]
        k.kv_pages_workspace_bytes.argtypes = [c_int, c_int]
        k.kv_pages_workspace_bytes.restype = c_size_t
        k.kv_pages_fork.argtypes = [c_void_p, c_size_t, c_int, c_int, c_size_t, c_int, c_void_p, c_int, c_void_p,
                                    c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p,
                                    c_void_p]
        k.kv_pages_compact.argtypes = [c_void_p, c_size_t, c_int, c_int, c_size_t, c_int, c_void_p, c_int, c_void_p,
                                       c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p, c_void_p]
        _lib = k
    return _lib


def kv4_cache(num_pages: int, nkv: int, device):
    """An empty 4-bit K or V cache, uint8 [pages][nkv][1152]."""
    import torch
    return torch.zeros(num_pages, nkv, PAGE4_BYTES, dtype=torch.uint8, device=device)


def _check_kv4(k_cache, v_cache):
    shape = k_cache.shape
    if len(shape) != 3 or shape[2] != PAGE4_BYTES or k_cache.element_size() != 1 or v_cache.element_size() != 1 or \
            not k_cache.is_contiguous() or not v_cache.is_contiguous() or v_cache.shape != shape:
        raise ValueError(f"k_cache and v_cache are contiguous uint8 tensors [pages][nkv][{PAGE4_BYTES}]")


def _check_page_table(page_table, rows, row_seq):
    """Two dimensions, and where rows map to themselves one row each."""
    if page_table.dim() != 2:
        raise ValueError("the page table is a tensor [sequences][pages]")
    if row_seq is None and page_table.shape[0] < rows:
        raise ValueError("the page table has a row per row of the call when row_seq is None")


def _check_workspace(workspace):
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous")


@functools.lru_cache(maxsize=1024)
def _splits(B: int, nq: int, nkv: int, max_context: int, split_tokens: int | None, max_splits: int | None):
    """(tokens of a split, splits, workspace bytes)."""
    split = lib().attn_kv4_split_tokens(B, nkv, max_context) if split_tokens is None else split_tokens
    if split <= 0:
        raise ValueError("split_tokens is positive")
    n = -(-max_context // split) if max_splits is None else max_splits
    return split, n, max(lib().attn_kv4_decode_workspace_bytes(B, nq, n), 16)


@functools.lru_cache(maxsize=1024)
def _pages_workspace(pages: int, rows: int) -> int:
    return lib().kv_pages_workspace_bytes(pages, rows)


def kv4_rope_write(qkv, positions, row_seq, page_table, k_cache, v_cache, nq: int, rot: int, inv_freq,
                   keys: bool = False, seq_lens_out=None, error_word=None, stream=None):
    """attn_kv4_rope_write_rows: qkv bf16 [B][(nq + 2 nkv) * 128] -> (rotated q bf16 [B][nq][128], with `keys` the
    rotated keys bf16 [B][nkv][128] before quantisation, else None); k and v into their page slots.  row_seq None:
    row b uses page-table row b."""
    import torch
    _check_kv4(k_cache, v_cache)
    A.check_rows("qkv", qkv, torch.bfloat16, (nq + 2 * k_cache.shape[1]) * HEAD_DIM)
    A.check_i32(positions, row_seq, page_table, seq_lens_out, error_word)
    B = qkv.shape[0]
    if positions.numel() != B or (B if row_seq is None else row_seq.numel()) != B or \
            (B if seq_lens_out is None else seq_lens_out.numel()) != B:
        raise ValueError("positions, row_seq and seq_lens_out have one entry per row")
    if inv_freq is not None and (inv_freq.numel() < rot // 2 or inv_freq.dtype is not torch.float32 or
                                 not inv_freq.is_contiguous()):
        raise ValueError("inv_freq has rot / 2 contiguous float32 entries")
    _check_page_table(page_table, B, row_seq)
    return A.on_stream(qkv, stream, _rope_write, qkv, positions, row_seq, page_table, k_cache, v_cache, nq, rot, inv_freq,
                       keys, seq_lens_out, error_word)


def _rope_write(stream, qkv, positions, row_seq, page_table, k_cache, v_cache, nq, rot, inv_freq, keys, seq_lens_out,
                error_word):
    import torch
    B, (pages, nkv, _) = qkv.shape[0], k_cache.shape
    q = torch.empty(B, nq, HEAD_DIM, dtype=torch.bfloat16, device=qkv.device)
    k = torch.empty(B, nkv, HEAD_DIM, dtype=torch.bfloat16, device=qkv.device) if keys else None
    M.check("attn_kv4_rope_write_rows", lib().attn_kv4_rope_write_rows(
        qkv.data_ptr(), B, nq, nkv, HEAD_DIM, rot, M.ptr(inv_freq), positions.data_ptr(), M.ptr(row_seq),
        page_table.shape[0], page_table.data_ptr(), page_table.shape[1], PAGE, pages, q.data_ptr(), M.ptr(k),
        k_cache.data_ptr(), v_cache.data_ptr(), M.ptr(seq_lens_out), M.ptr(error_word), stream))
    return q, k


def kv4_read_rows(k_cache, v_cache, positions, row_seq, page_table, error_word=None, stream=None):
    """attn_kv4_read_rows: the tokens at `positions` of page-table rows `row_seq` as the bf16 values the cache holds:
    (k, v), each [B][nkv][128]."""
    _check_kv4(k_cache, v_cache)
    A.check_i32(positions, row_seq, page_table, error_word)
    B = positions.numel()
    if row_seq is not None and row_seq.numel() != B:
        raise ValueError("row_seq has one entry per position")
    _check_page_table(page_table, B, row_seq)
    return A.on_stream(k_cache, stream, _read_rows, k_cache, v_cache, positions, row_seq, page_table, error_word)


def _read_rows(stream, k_cache, v_cache, positions, row_seq, page_table, error_word):
    import torch
    B, (pages, nkv, _) = positions.numel(), k_cache.shape
    k = torch.empty(B, nkv, HEAD_DIM, dtype=torch.bfloat16, device=k_cache.device)
    v = torch.empty_like(k)
    M.check("attn_kv4_read_rows", lib().attn_kv4_read_rows(
        k_cache.data_ptr(), v_cache.data_ptr(), pages, positions.data_ptr(), M.ptr(row_seq), page_table.shape[0],
        page_table.data_ptr(), page_table.shape[1], PAGE, B, nkv, HEAD_DIM, k.data_ptr(), v.data_ptr(), M.ptr(error_word),
        stream))
    return k, v


def kv4_decode(q, k_cache, v_cache, page_table, seq_lens, scale: float, row_seq=None, split_tokens: int | None = None,
               max_splits: int | None = None, quant: bool = False, workspace=None, error_word=None, stream=None):
    """attn_kv4_decode_rows: attention of q bf16 [B][nq][128] over the first seq_lens[b] tokens of page-table row
    row_seq[b] (None: b).  split_tokens None: the split that fills the GPU if contexts are as long as the page table is wide;
    under a table much wider than they are, give split_tokens and max_splits (attn_kv4_split_tokens of the longest context
    on hand).  Returns (out bf16 [B][nq][128], out_q e4m3
    [B][nq * 128] or None, out_s [nq][ld] or None)."""
    import torch
    _check_kv4(k_cache, v_cache)
    A.check_heads("q", q, torch.bfloat16)
    A.check_i32(page_table, seq_lens, row_seq, error_word)
    if not q.is_contiguous():
        raise ValueError("q is contiguous")
    B = q.shape[0]
    if seq_lens.numel() != B or (B if row_seq is None else row_seq.numel()) != B:
        raise ValueError("seq_lens and row_seq have one entry per row of q")
    _check_page_table(page_table, B, row_seq)
    _check_workspace(workspace)
    return A.on_stream(q, stream, _decode, q, k_cache, v_cache, page_table, seq_lens, scale, row_seq, split_tokens,
                       max_splits, quant, workspace, error_word)


def _decode(stream, q, k_cache, v_cache, page_table, seq_lens, scale, row_seq, split_tokens, max_splits, quant, workspace,
            error_word):
    import torch
    (B, nq, _), (pages, nkv, _), (num_seqs, max_pages) = q.shape, k_cache.shape, page_table.shape
    split_tokens, max_splits, need = _splits(B, nq, nkv, max_pages * PAGE, split_tokens, max_splits)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    out = torch.empty_like(q)
    out_q = out_s = None
    ld = (B + 3) // 4 * 4
    if quant:
        out_q = torch.empty(B, nq * HEAD_DIM, dtype=torch.uint8, device=q.device)
        out_s = torch.empty(nq, ld, dtype=torch.float32, device=q.device)
    M.check("attn_kv4_decode_rows", lib().attn_kv4_decode_rows(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pages, page_table.data_ptr(), max_pages, M.ptr(row_seq),
        num_seqs, seq_lens.data_ptr(), B, nq, nkv, HEAD_DIM, PAGE, scale, split_tokens, max_splits, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), out.data_ptr(), M.ptr(out_q), M.ptr(out_s), ld, M.ptr(error_word),
        stream))
    return out, out_q, out_s


# ---------------------------------------------------------------- pages

def _cache_args(caches):
    """(pointer, bytes between caches, caches, pages, bytes of a page) of a tensor [caches][pages][...]."""
    shape, stride, e = caches.shape, caches.stride(), caches.element_size()
    inner = 1
    for n, st in zip(reversed(shape[1:]), reversed(stride[1:])):
        if n != 1 and st != inner:
            raise ValueError("caches is a tensor [caches][pages][...] with every cache contiguous")
        inner *= n
    if len(shape) < 3:
        raise ValueError("caches is a tensor [caches][pages][...] with every cache contiguous")
    return caches.data_ptr(), stride[0] * e, shape[0], shape[1], inner // max(shape[1], 1) * e


def _check_table(table, lens):
    if table.dim() != 2 or lens.numel() != table.shape[0]:
        raise ValueError("the page table is a tensor [sequences][pages] and lens has one entry per row of it")


def fork_pages(caches, table, lens, parents, reserve=None, workspace=None, error_word=None, stream=None):
    """kv_pages_fork: row i of the result is row parents[i] (-1: empty) with room for reserve[i] more tokens; full
    pages are shared, a page in part filled is copied for all appending rows but one.  Returns (table, lens) int32,
    new tensors."""
    A.check_i32(table, lens, parents, reserve, error_word)
    _check_table(table, lens)
    _check_workspace(workspace)
    if reserve is not None and reserve.numel() != parents.numel():
        raise ValueError("reserve has one entry per parent")
    return A.on_stream(caches, stream, _fork, caches, table, lens, parents, reserve, workspace, error_word)


def _fork(stream, caches, table, lens, parents, reserve, workspace, error_word):
    import torch
    ptr, stride, n, pages, page_bytes = _cache_args(caches)
    rows, max_pages = parents.numel(), table.shape[1]
    if workspace is None:
        workspace = torch.empty(_pages_workspace(pages, rows), dtype=torch.uint8, device=caches.device)
    out = torch.empty(rows, max_pages, dtype=torch.int32, device=caches.device)
    lens_out = torch.empty(rows, dtype=torch.int32, device=caches.device)
    M.check("kv_pages_fork", lib().kv_pages_fork(
        ptr, stride, n, pages, page_bytes, PAGE, table.data_ptr(), max_pages, lens.data_ptr(), table.shape[0],
        parents.data_ptr(), M.ptr(reserve), rows, out.data_ptr(), lens_out.data_ptr(), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), M.ptr(error_word), stream))
    return out, lens_out


def compact_pages(caches, table, lens, out=None, workspace=None, error_word=None, stream=None):
    """kv_pages_compact: moves the pages in use to the lowest ids.  Returns (table, pages in use int32 [1]); `out` may
    be `table` itself."""
    A.check_i32(table, lens, out, error_word)
    _check_table(table, lens)
    _check_workspace(workspace)
    if out is not None and out.shape != table.shape:
        raise ValueError("out has the page table's shape")
    return A.on_stream(caches, stream, _compact, caches, table, lens, out, workspace, error_word)


def _compact(stream, caches, table, lens, out, workspace, error_word):
    import torch
    ptr, stride, n, pages, page_bytes = _cache_args(caches)
    seqs, max_pages = table.shape
    if workspace is None:
        workspace = torch.empty(_pages_workspace(pages, seqs), dtype=torch.uint8, device=caches.device)
    out = torch.empty_like(table) if out is None else out
    used = torch.empty(1, dtype=torch.int32, device=caches.device)
    M.check("kv_pages_compact", lib().kv_pages_compact(
        ptr, stride, n, pages, page_bytes, PAGE, table.data_ptr(), max_pages, lens.data_ptr(), seqs, out.data_ptr(),
        used.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(), M.ptr(error_word), stream))
    return out, used
