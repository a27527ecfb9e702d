"""Linear layer over weights held in 4 bits, beside the bitmap one: for matrices that are quantised instead of pruned.

Weight (m, k) is s (c - z): code c and zero point z in 0..15, scale s fp16, both shared by 32, 64 or 128 consecutive k.
"""
from dataclasses import dataclass

import torch

from . import _lib
from .api import ACT_NONE, SpmmError, _check, _hand_over, _on, _ptr, _raw, _stream_ptr


@dataclass
class Int4Matrix:
    """A weight matrix resident on the GPU in the library's 4-bit layout."""
    M: int
    K: int
    group: int
    data: torch.Tensor   # uint8: codes, scales and zero points of 128 x 128 pieces, M and K rounded up to 128

    def algorithmic_bytes(self, N):
        """Bytes one linear_int4 must move: codes, scales and zero points, activations, output."""
        return self.data.numel() + 2 * self.K * N + 2 * self.M * N


def _shape(M, K, group):
    if M <= 0 or K <= 0 or M % 64 or K % 64:
        raise SpmmError("M and K must be positive multiples of 64")
    if group not in (32, 64, 128) or K % group:
        raise SpmmError("the group must be 32, 64 or 128 and divide K")


def _need(t, name, dtype, shape, device=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.is_contiguous() and tuple(t.shape) == tuple(shape)
            and (device is None or t.device == device)):
        raise SpmmError(f"{name} must be a contiguous CUDA {str(dtype).split('.')[1]} {list(shape)} tensor"
                        + (f" on {device}" if device is not None else ""))


def pack_int4(codes, scales, zeros, stream=None):
    """codes uint8 [M, K] (0..15), scales float16 [M, K/group], zeros uint8 [M, K/group] (0..15), as quantisation tools deliver
    them -> Int4Matrix.  Only the low four bits of codes and zero points are used."""
    if codes.dim() != 2 or scales.dim() != 2 or scales.shape[1] <= 0 or codes.shape[1] % scales.shape[1]:
        raise SpmmError("codes must be [M, K] and scales [M, K/group]")
    M, K = codes.shape
    group = K // scales.shape[1]
    _shape(M, K, group)
    _need(codes, "codes", torch.uint8, (M, K))
    _need(scales, "scales", torch.float16, (M, K // group), codes.device)
    _need(zeros, "zeros", torch.uint8, (M, K // group), codes.device)
    with _on(codes.device, stream):
        data = torch.empty(_lib.load().spb_int4_bytes(M, K, group), dtype=torch.uint8, device=codes.device)
        _check(_lib.load().spb_int4_pack(_stream_ptr(stream), _ptr(codes), _ptr(scales), _ptr(zeros), M, K, group, _ptr(data)),
               "spb_int4_pack")
    return Int4Matrix(M, K, group, _hand_over(data, stream))


def encode_int4(A, group=128, stream=None):
    """Quantise a dense CUDA float16 matrix [M, K] to the nearest codes of a range that holds zero -> Int4Matrix."""
    if not (A.is_cuda and A.dtype == torch.float16 and A.dim() == 2 and A.is_contiguous()):
        raise SpmmError("A must be a contiguous CUDA float16 matrix")
    M, K = A.shape
    _shape(M, K, group)
    with _on(A.device, stream):
        codes = torch.empty((M, K), dtype=torch.uint8, device=A.device)
        scales = torch.empty((M, K // group), dtype=torch.float16, device=A.device)
        zeros = torch.empty((M, K // group), dtype=torch.uint8, device=A.device)
        _check(_lib.load().spb_int4_encode(_stream_ptr(stream), _ptr(A), M, K, group, _ptr(codes), _ptr(scales), _ptr(zeros)), "spb_int4_encode")
    return pack_int4(codes, scales, zeros, stream)


def _check_matrix(W):
    _shape(W.M, W.K, W.group)
    _need(W.data, "W.data", torch.uint8, (_lib.load().spb_int4_bytes(W.M, W.K, W.group),))


def decode_int4(W: Int4Matrix, out=None, stream=None):
    """The dense fp16 matrix [M, K] that W stands for, s (c - z) rounded once."""
    _check_matrix(W)
    if out is not None:
        _need(out, "out", torch.float16, (W.M, W.K), W.data.device)
    with _on(W.data.device, stream):
        y = out if out is not None else torch.empty((W.M, W.K), dtype=torch.float16, device=W.data.device)
        _check(_lib.load().spb_int4_decode(_stream_ptr(stream), _ptr(W.data), W.M, W.K, W.group, _ptr(y)), "spb_int4_decode")
    return out if out is not None else _hand_over(y, stream)


def int4_workspace(W, N):
    """Bytes of the workspace `linear_int4` needs for N rows (0 for many shapes)."""
    with torch.cuda.device(W.data.device):
        return _lib.load().spb_int4_workspace_bytes(W.M, N, W.K)


def linear_int4(W: Int4Matrix, B, bias=None, residual=None, activation=ACT_NONE, out=None, workspace=None, stream=None):
    """spb_linear_int4: out[N,M] = residual + act(B W^T + bias), summed in fp32 and rounded to fp16 once.  B [N,K] as in
    `linear`; out may be the residual itself, not B.  workspace: int4_workspace(W, N) bytes; a new one by default."""
    return _lib.ext().linear_int4(W.data, W.M, W.K, W.group, B, bias, residual, activation, out, workspace, _raw(stream, W.data.device))
