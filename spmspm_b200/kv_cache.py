"""Paged key/value cache in 4 bits and attention over it.

32 consecutive channels of a token and head are held as m + s c (m, s fp16, c in 0..15): 5 bits a channel instead of 16.  Every call
describes its batch with the same three device tensors, so that a captured step keeps working while the contexts grow:

    page_table  int32 [batch, pages]   page that holds tokens i * page_size .. of a sequence (-1: none)
    kv_lens     int32 [batch]          tokens of the sequence in the cache, those of this call included
    cu_q        int32 [batch + 1]      rows cu_q[b] .. cu_q[b + 1] - 1 of the packed inputs are the last tokens of sequence b;
                                       None: the same number for every sequence

A page number outside the pool or a token past the table sets bit 8 of `device_status()`.
"""
import torch

from . import _lib
from .api import SpmmError, _raw


class KvCacheInt4:
    """The pool: num_pages pages of page_size tokens (a multiple of 16) for kv_heads heads of 64 or 128 channels."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        if head_dim not in (64, 128):
            raise SpmmError("head_dim must be 64 or 128")
        if num_pages <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % 16 or page_size > 65536:
            raise SpmmError("num_pages and kv_heads must be positive, page_size a multiple of 16 up to 65536")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = int(num_pages), int(page_size), int(kv_heads), int(head_dim)
        self._pool = torch.zeros(_lib.load().spb_kv_cache_bytes(num_pages, page_size, kv_heads, head_dim), dtype=torch.uint8, device=device)
        if not self._pool.is_cuda:
            raise SpmmError("the cache lives on a CUDA device")
        self._open()

    def _open(self):
        self._handle = _lib.ext().Cache(self._pool, self.num_pages, self.page_size, self.kv_heads, self.head_dim)

    @property
    def pool(self):
        """The pages, uint8."""
        return self._pool

    def __getstate__(self):   # copies and saved caches have a handle of their own
        return {k: v for k, v in self.__dict__.items() if k != "_handle"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._open()

    def token_bytes(self):
        """Bytes a token takes in one layer: codes, scales and minima of keys and values of all heads."""
        return self.kv_heads * 20 * self.head_dim // 16


def kv_append(cache, k, v, page_table, kv_lens, cu_q=None, q=None, cos=None, sin=None, interleaved=False, q_out=None, stream=None):
    """spb_kv_append: write the keys and values [tokens, kv_heads, head_dim] of the new tokens.

    With cos and sin (float32 [positions, rot/2]) the first rot channels of the keys are first turned by the angles of the
    token's position in the cache, and so are those of q [tokens, heads, head_dim], which is returned (q_out, which may be q itself,
    or a new tensor).
    Tokens before the start of the context or past the angles are skipped as a whole; their rows, and those of no sequence, leave q_out as
    it was (a new tensor has no defined value there)."""
    return _lib.ext().kv_append(cache._handle, k, v, page_table, kv_lens, cu_q, q, cos, sin, interleaved, q_out, _raw(stream, cache.pool.device))


def kv_read(cache, page_table, kv_lens, cu_q=None, n_tokens=None, k_out=None, v_out=None, stream=None):
    """spb_kv_read: k, v [n_tokens, kv_heads, head_dim] fp16, what the cache holds for the last tokens of every sequence (n_tokens is
    the number of packed rows, cu_q[-1] on the host; it may be left out when k_out is given)."""
    return _lib.ext().kv_read(cache._handle, page_table, kv_lens, cu_q, n_tokens, k_out, v_out, _raw(stream, cache.pool.device))


def kv_attention_workspace(cache, q_heads, batch, max_q):
    """Bytes of the workspace `kv_attention` needs for such a call."""
    return _lib.ext().kv_attention_workspace(cache._handle, q_heads, batch, max_q)


def kv_attention(q, cache, page_table, kv_lens, cu_q=None, max_q=None, scale=None, out=None, workspace=None, stream=None):
    """spb_kv_attention: out [tokens, heads, head_dim] = softmax(scale q K^T) V over the keys of the row's sequence up to its own position.

    max_q: an upper bound of the new tokens of one sequence (default: tokens / batch without cu_q, all of them with it); it
    chooses the kernel only.  With cu_q it should be given: many sequences with few new tokens each are else taken for a prompt.  scale: 1 / sqrt(head_dim) by default.  out may be q itself.  workspace: kv_attention_workspace() bytes; a new one
    by default.  Rows that see no key get zeros, rows that belong to no sequence are left as they were."""
    return _lib.ext().kv_attention(q, cache._handle, page_table, kv_lens, cu_q, max_q, scale, out, workspace, _raw(stream, cache.pool.device))
