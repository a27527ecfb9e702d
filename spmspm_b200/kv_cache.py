"""Paged key/value cache in 4 bits and attention over it.

32 consecutive channels of a token and head are held as m + s c (m, s fp16, c in 0..15): 5 bits a channel instead of 16.  Every call
describes its batch with the same three device tensors, so that a captured step keeps working while the contexts grow:

    page_table  int32 [batch, pages]   page that holds tokens i * page_size .. of a sequence (-1: none)
    kv_lens     int32 [batch]          tokens of the sequence in the cache, those of this call included
    cu_q        int32 [batch + 1]      rows cu_q[b] .. cu_q[b + 1] - 1 of the packed inputs are the last tokens of sequence b;
                                       None: the same number for every sequence

A page number outside the pool or a token past the table sets bit 8 of `device_status()`.
"""
import ctypes
import math

import torch

from . import _lib
from .api import SpmmError, _check, _ptr, _stream_ptr


class KvCacheInt4:
    """The pool: num_pages pages of page_size tokens (a multiple of 16) for kv_heads heads of 64 or 128 channels."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        if head_dim not in (64, 128):
            raise SpmmError("head_dim must be 64 or 128")
        if num_pages <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % 16 or page_size > 65536:
            raise SpmmError("num_pages and kv_heads must be positive, page_size a multiple of 16 up to 65536")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = int(num_pages), int(page_size), int(kv_heads), int(head_dim)
        self.pool = torch.zeros(_lib.load().spb_kv_cache_bytes(num_pages, page_size, kv_heads, head_dim), dtype=torch.uint8, device=device)

    def token_bytes(self):
        """Bytes a token takes in one layer: codes, scales and minima of keys and values of all heads."""
        return self.kv_heads * 20 * self.head_dim // 16


def _batch(cache, page_table, kv_lens, cu_q):
    dev = cache.pool.device
    if not (page_table.is_cuda and page_table.device == dev and page_table.dtype == torch.int32 and page_table.dim() == 2
            and page_table.stride(1) == 1 and page_table.shape[0] > 0 and page_table.shape[1] > 0
            and page_table.stride(0) == page_table.shape[1]):
        raise SpmmError("page_table must be a contiguous CUDA int32 [batch, pages] tensor on the cache's device")
    batch = page_table.shape[0]
    for name, t, n in (("kv_lens", kv_lens, batch), ("cu_q", cu_q, batch + 1)):
        if t is not None and not (t.is_cuda and t.device == dev and t.dtype == torch.int32 and t.is_contiguous() and tuple(t.shape) == (n,)):
            raise SpmmError(f"{name} must be a contiguous CUDA int32 [{n}] tensor on the cache's device")
    if kv_lens is None:
        raise SpmmError("kv_lens is missing")
    return batch


def _vectors(cache, t, name, heads, n=None):
    """[tokens, heads, head_dim] with contiguous channels; strides that hold four channels together."""
    if not (t.is_cuda and t.device == cache.pool.device and t.dtype == torch.float16 and t.dim() == 3 and t.shape[2] == cache.head_dim
            and (heads is None or t.shape[1] == heads) and (n is None or t.shape[0] == n)):
        raise SpmmError(f"{name} must be a CUDA float16 [tokens, {'heads' if heads is None else heads}, {cache.head_dim}] tensor on the cache's device")
    if t.numel() and (t.stride(2) != 1 or t.stride(0) % 4 or t.stride(1) % 4 or t.data_ptr() % 8):
        raise SpmmError(f"{name} must have contiguous channels, strides that are multiples of 4 and an 8-byte aligned start")
    return t.stride(0), t.stride(1)


def _rows(n_tokens, batch, cu_q):
    if cu_q is None and n_tokens % batch:
        raise SpmmError("without cu_q the tokens must divide evenly among the sequences")


def _dense(t, name, shape, cache):
    if not (t.is_cuda and t.device == cache.pool.device and t.dtype == torch.float16 and t.is_contiguous() and tuple(t.shape) == tuple(shape)):
        raise SpmmError(f"{name} must be a contiguous CUDA float16 {list(shape)} tensor on the cache's device")
    return t


def _cache_args(cache, page_table, kv_lens, cu_q, batch, n):
    return (_ptr(cache.pool), cache.num_pages, cache.page_size, cache.kv_heads, cache.head_dim, _ptr(page_table), page_table.shape[1],
            _ptr(kv_lens), _ptr(cu_q), batch, n)


def kv_append(cache, k, v, page_table, kv_lens, cu_q=None, q=None, cos=None, sin=None, interleaved=False, q_out=None, stream=None):
    """spb_kv_append: write the keys and values [tokens, kv_heads, head_dim] of the new tokens.

    With cos and sin (float32 [positions, rot/2]) the first rot channels of the keys are first turned by the angles of the
    token's position in the cache, and so are those of q [tokens, heads, head_dim], which is returned (q_out, or a new tensor).
    Rows that belong to no sequence leave q_out as it was."""
    batch = _batch(cache, page_table, kv_lens, cu_q)
    ks = _vectors(cache, k, "k", cache.kv_heads)
    n = k.shape[0]
    vs = _vectors(cache, v, "v", cache.kv_heads, n)
    _rows(n, batch, cu_q)
    if (cos is None) != (sin is None):
        raise SpmmError("cos and sin are given together")
    rot = max_pos = 0
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if not (t.is_cuda and t.device == cache.pool.device and t.dtype == torch.float32 and t.dim() == 2 and t.is_contiguous()
                    and t.shape == cos.shape and t.shape[0] > 0):
                raise SpmmError(f"{name} must be a contiguous CUDA float32 [positions, rot/2] tensor on the cache's device")
        max_pos, rot = cos.shape[0], 2 * cos.shape[1]
        if rot == 0 or rot % 8 or rot > cache.head_dim:
            raise SpmmError("the rotated channels must be a multiple of 8 up to head_dim")
    if q is None and q_out is not None:
        raise SpmmError("q_out without q")
    qs, heads = (0, 0), 0
    if q is not None:
        if cos is None:
            raise SpmmError("q is only taken to be rotated: cos and sin are missing")
        qs = _vectors(cache, q, "q", None, n)
        heads = q.shape[1]
        if heads == 0:
            raise SpmmError("q has no heads")
        q_out = _dense(q_out, "q_out", q.shape, cache) if q_out is not None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if n:
        with torch.cuda.device(cache.pool.device):
            _check(_lib.load().spb_kv_append(_stream_ptr(stream), *_cache_args(cache, page_table, kv_lens, cu_q, batch, n), _ptr(k), *ks, _ptr(v), *vs,
                                             _ptr(q), *qs, heads, _ptr(q_out), _ptr(cos), _ptr(sin), max_pos, rot, int(bool(interleaved))),
                   "spb_kv_append")
    return q_out


def kv_read(cache, page_table, kv_lens, cu_q=None, n_tokens=None, k_out=None, v_out=None, stream=None):
    """spb_kv_read: k, v [n_tokens, kv_heads, head_dim] fp16, what the cache holds for the last tokens of every sequence (n_tokens is
    the number of packed rows, cu_q[-1] on the host; it may be left out when k_out is given)."""
    batch = _batch(cache, page_table, kv_lens, cu_q)
    if n_tokens is None:
        if k_out is None:
            raise SpmmError("n_tokens or k_out is needed")
        n_tokens = k_out.shape[0]
    if n_tokens < 0:
        raise SpmmError("n_tokens must not be negative")
    _rows(n_tokens, batch, cu_q)
    shape = (int(n_tokens), cache.kv_heads, cache.head_dim)
    k_out, v_out = (torch.empty(shape, dtype=torch.float16, device=cache.pool.device) if t is None else _dense(t, name, shape, cache)
                    for name, t in (("k_out", k_out), ("v_out", v_out)))
    if n_tokens:
        with torch.cuda.device(cache.pool.device):
            _check(_lib.load().spb_kv_read(_stream_ptr(stream), *_cache_args(cache, page_table, kv_lens, cu_q, batch, int(n_tokens)), _ptr(k_out),
                                           _ptr(v_out)), "spb_kv_read")
    return k_out, v_out


def kv_attention_workspace(cache, q_heads, batch, max_q):
    """Bytes of the workspace `kv_attention` needs for such a call."""
    with torch.cuda.device(cache.pool.device):
        return _lib.load().spb_kv_attention_workspace_bytes(cache.head_dim, batch, q_heads, cache.kv_heads, max_q)


def kv_attention(q, cache, page_table, kv_lens, cu_q=None, max_q=None, scale=None, out=None, workspace=None, stream=None):
    """spb_kv_attention: out [tokens, heads, head_dim] = softmax(scale q K^T) V over the keys of the row's sequence up to its own position.

    max_q: an upper bound of the new tokens of one sequence (default: tokens / batch without cu_q, all of them with it); it
    chooses the tiling only.  scale: 1 / sqrt(head_dim) by default.  workspace: uint8, kv_attention_workspace() bytes; a new one
    by default.  Rows that see no key get zeros, rows that belong to no sequence are left as they were."""
    batch = _batch(cache, page_table, kv_lens, cu_q)
    qs = _vectors(cache, q, "q", None)
    n, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise SpmmError("the heads of q must be a positive multiple of the cache's")
    _rows(n, batch, cu_q)
    if max_q is None:
        max_q = n if cu_q is not None else n // batch
    if max_q < 0 or max_q > n:
        raise SpmmError("max_q must be in 0..tokens")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else _dense(out, "out", q.shape, cache)
    if not n:
        return out
    need = kv_attention_workspace(cache, heads, batch, int(max_q))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        if stream is not None:
            workspace.record_stream(stream)   # its memory must not go to another tensor before that stream is done with it
    elif not (workspace.is_cuda and workspace.device == q.device and workspace.is_contiguous()
              and workspace.numel() * workspace.element_size() >= need):
        raise SpmmError(f"the workspace must be a contiguous CUDA tensor of at least {need} bytes on the cache's device")
    with torch.cuda.device(cache.pool.device):
        _check(_lib.load().spb_kv_attention(_stream_ptr(stream), *_cache_args(cache, page_table, kv_lens, cu_q, batch, n), _ptr(q), *qs, heads,
                                            int(max_q), ctypes.c_float(1 / math.sqrt(cache.head_dim) if scale is None else float(scale)), _ptr(out),
                                            _ptr(workspace), workspace.numel() * workspace.element_size()), "spb_kv_attention")
    return out
