"""Paged key/value cache in 4 bits and attention over it.

32 consecutive channels of a token and head are held as m + s c (m, s fp16, c in 0..15): 5 bits a channel instead of 16.  Every call
describes its batch with the same three device tensors, so that a captured step keeps working while the contexts grow:

    page_table  int32 [batch, pages]   page that holds tokens i * page_size .. of a sequence (-1: none)
    kv_lens     int32 [batch]          tokens of the sequence in the cache, those of this call included
    cu_q        int32 [batch + 1]      rows cu_q[b] .. cu_q[b + 1] - 1 of the packed inputs are the last tokens of sequence b;
                                       None: the same number for every sequence

A page number outside the pool or a token past the table sets bit 8 of `device_status()`.
"""
import functools
import math

import torch

from . import _lib
from .api import SpmmError, _call


class KvCacheInt4:
    """The pool: num_pages pages of page_size tokens (a multiple of 16) for kv_heads heads of 64 or 128 channels."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        if head_dim not in (64, 128):
            raise SpmmError("head_dim must be 64 or 128")
        if num_pages <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % 16 or page_size > 65536:
            raise SpmmError("num_pages and kv_heads must be positive, page_size a multiple of 16 up to 65536")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = int(num_pages), int(page_size), int(kv_heads), int(head_dim)
        self.pool = torch.zeros(_lib.load().spb_kv_cache_bytes(num_pages, page_size, kv_heads, head_dim), dtype=torch.uint8, device=device)
        if not self.pool.is_cuda:
            raise SpmmError("the cache lives on a CUDA device")

    def token_bytes(self):
        """Bytes a token takes in one layer: codes, scales and minima of keys and values of all heads."""
        return self.kv_heads * 20 * self.head_dim // 16


# The checks run on every call of a decode step, whose kernels take a few microseconds: they read each attribute once, and the
# device and stream are looked up as integers.

def _batch(cache, dev, page_table, kv_lens, cu_q):
    """Checks the tensors that describe the batch; the arguments of the library that name the cache and the batch."""
    shape = page_table.shape
    if page_table.get_device() != dev or page_table.dtype is not torch.int32 or len(shape) != 2 or not page_table.is_contiguous() or 0 in shape:
        raise SpmmError("page_table must be a contiguous CUDA int32 [batch, pages] tensor on the cache's device")
    batch, width = shape
    if kv_lens is None or kv_lens.get_device() != dev or kv_lens.dtype is not torch.int32 or kv_lens.shape != (batch,) or not kv_lens.is_contiguous():
        raise SpmmError(f"kv_lens must be a contiguous CUDA int32 [{batch}] tensor on the cache's device")
    cu = None
    if cu_q is not None:
        if cu_q.get_device() != dev or cu_q.dtype is not torch.int32 or cu_q.shape != (batch + 1,) or not cu_q.is_contiguous():
            raise SpmmError(f"cu_q must be a contiguous CUDA int32 [{batch + 1}] tensor on the cache's device")
        cu = cu_q.data_ptr()
    return batch, (cache.pool.data_ptr(), cache.num_pages, cache.page_size, cache.kv_heads, cache.head_dim, page_table.data_ptr(), width,
                   kv_lens.data_ptr(), cu, batch)


def _vectors(cache, dev, t, name, heads=None, n=None):
    """[tokens, heads, head_dim] with contiguous channels and strides that hold four channels together: shape, address, strides."""
    shape = t.shape
    if (t.get_device() != dev or t.dtype is not torch.float16 or len(shape) != 3 or shape[2] != cache.head_dim
            or (heads is not None and shape[1] != heads) or (n is not None and shape[0] != n)):
        raise SpmmError(f"{name} must be a CUDA float16 [{'tokens' if n is None else n}, {'heads' if heads is None else heads}, {cache.head_dim}] "
                        "tensor on the cache's device")
    tok, head, ch = t.stride()
    at = t.data_ptr()
    if (ch != 1 or (tok | head) & 3 or at & 7) and t.numel():
        raise SpmmError(f"{name} must have contiguous channels, strides that are multiples of 4 and an 8-byte aligned start")
    return shape, at, tok, head


def _rows(n_tokens, batch, cu_q):
    if cu_q is None and n_tokens % batch:
        raise SpmmError("without cu_q the tokens must divide evenly among the sequences")


def _dense(t, name, shape, dev):
    if t.get_device() != dev or t.dtype is not torch.float16 or not t.is_contiguous() or t.shape != shape:
        raise SpmmError(f"{name} must be a contiguous CUDA float16 {list(shape)} tensor on the cache's device")
    return t


def kv_append(cache, k, v, page_table, kv_lens, cu_q=None, q=None, cos=None, sin=None, interleaved=False, q_out=None, stream=None):
    """spb_kv_append: write the keys and values [tokens, kv_heads, head_dim] of the new tokens.

    With cos and sin (float32 [positions, rot/2]) the first rot channels of the keys are first turned by the angles of the
    token's position in the cache, and so are those of q [tokens, heads, head_dim], which is returned (q_out, or a new tensor).
    Rows that belong to no sequence leave q_out as it was."""
    dev = cache.pool.get_device()
    batch, args = _batch(cache, dev, page_table, kv_lens, cu_q)
    shape, k_at, k_tok, k_head = _vectors(cache, dev, k, "k", cache.kv_heads)
    n = shape[0]
    _, v_at, v_tok, v_head = _vectors(cache, dev, v, "v", cache.kv_heads, n)
    _rows(n, batch, cu_q)
    if (cos is None) != (sin is None):
        raise SpmmError("cos and sin are given together")
    rot = max_pos = 0
    cos_at = sin_at = None
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.get_device() != dev or t.dtype is not torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.shape != cos.shape or not t.shape[0]:
                raise SpmmError(f"{name} must be a contiguous CUDA float32 [positions, rot/2] tensor on the cache's device")
        max_pos, rot = cos.shape[0], 2 * cos.shape[1]
        if rot == 0 or rot % 8 or rot > cache.head_dim:
            raise SpmmError("the rotated channels must be a multiple of 8 up to head_dim")
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    if q is None:
        if q_out is not None:
            raise SpmmError("q_out without q")
        heads = q_tok = q_head = 0
        q_at = out_at = None
    else:
        if cos is None:
            raise SpmmError("q is only taken to be rotated: cos and sin are missing")
        q_shape, q_at, q_tok, q_head = _vectors(cache, dev, q, "q", None, n)
        heads = q_shape[1]
        if heads == 0:
            raise SpmmError("q has no heads")
        q_out = torch.empty(q_shape, dtype=torch.float16, device=q.device) if q_out is None else _dense(q_out, "q_out", q_shape, dev)
        out_at = q_out.data_ptr()
    if n:
        _call("spb_kv_append", dev, stream, *args, n, k_at, k_tok, k_head, v_at, v_tok, v_head, q_at, q_tok, q_head, heads, out_at, cos_at, sin_at,
              max_pos, rot, 1 if interleaved else 0)
    return q_out


def kv_read(cache, page_table, kv_lens, cu_q=None, n_tokens=None, k_out=None, v_out=None, stream=None):
    """spb_kv_read: k, v [n_tokens, kv_heads, head_dim] fp16, what the cache holds for the last tokens of every sequence (n_tokens is
    the number of packed rows, cu_q[-1] on the host; it may be left out when k_out is given)."""
    dev = cache.pool.get_device()
    batch, args = _batch(cache, dev, page_table, kv_lens, cu_q)
    if n_tokens is None:
        if k_out is None:
            raise SpmmError("n_tokens or k_out is needed")
        n_tokens = k_out.shape[0]
    n_tokens = int(n_tokens)
    if n_tokens < 0:
        raise SpmmError("n_tokens must not be negative")
    _rows(n_tokens, batch, cu_q)
    shape = (n_tokens, cache.kv_heads, cache.head_dim)
    k_out = torch.empty(shape, dtype=torch.float16, device=cache.pool.device) if k_out is None else _dense(k_out, "k_out", shape, dev)
    v_out = torch.empty(shape, dtype=torch.float16, device=cache.pool.device) if v_out is None else _dense(v_out, "v_out", shape, dev)
    if n_tokens:
        _call("spb_kv_read", dev, stream, *args, n_tokens, k_out.data_ptr(), v_out.data_ptr())
    return k_out, v_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev, head_dim, batch, q_heads, kv_heads, max_q):
    with torch.cuda.device(dev):
        return _lib.load().spb_kv_attention_workspace_bytes(head_dim, batch, q_heads, kv_heads, max_q)


def kv_attention_workspace(cache, q_heads, batch, max_q):
    """Bytes of the workspace `kv_attention` needs for such a call."""
    return _workspace_bytes(cache.pool.get_device(), cache.head_dim, batch, q_heads, cache.kv_heads, max_q)


def kv_attention(q, cache, page_table, kv_lens, cu_q=None, max_q=None, scale=None, out=None, workspace=None, stream=None):
    """spb_kv_attention: out [tokens, heads, head_dim] = softmax(scale q K^T) V over the keys of the row's sequence up to its own position.

    max_q: an upper bound of the new tokens of one sequence (default: tokens / batch without cu_q, all of them with it); it
    chooses the tiling only.  scale: 1 / sqrt(head_dim) by default.  workspace: kv_attention_workspace() bytes; a new one
    by default.  Rows that see no key get zeros, rows that belong to no sequence are left as they were."""
    dev = cache.pool.get_device()
    batch, args = _batch(cache, dev, page_table, kv_lens, cu_q)
    shape, q_at, q_tok, q_head = _vectors(cache, dev, q, "q")
    n, heads, d = shape
    if heads == 0 or heads % cache.kv_heads:
        raise SpmmError("the heads of q must be a positive multiple of the cache's")
    _rows(n, batch, cu_q)
    if max_q is None:
        max_q = n if cu_q is not None else n // batch
    if max_q < 0 or max_q > n:
        raise SpmmError("max_q must be in 0..tokens")
    out = torch.empty(shape, dtype=torch.float16, device=q.device) if out is None else _dense(out, "out", shape, dev)
    if not n:
        return out
    need = _workspace_bytes(dev, d, batch, heads, cache.kv_heads, max_q)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        if stream is not None:
            workspace.record_stream(stream)   # its memory must not go to another tensor before that stream is done with it
        have = need
    else:
        have = workspace.numel() * workspace.element_size()
        if workspace.get_device() != dev or not workspace.is_contiguous() or have < need:
            raise SpmmError(f"the workspace must be a contiguous CUDA tensor of at least {need} bytes on the cache's device")
    _call("spb_kv_attention", dev, stream, *args, n, q_at, q_tok, q_head, heads, max_q, 1 / math.sqrt(d) if scale is None else float(scale),
          out.data_ptr(), workspace.data_ptr(), have)
    return out
