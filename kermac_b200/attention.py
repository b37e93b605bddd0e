"""`cross_attention`, its gradient, and `prefix_attention`: kernel products with normalised weights.

Additive to the reference API.  `kernel_matvec` answers with y = K(b, a) c; here every row of K is exp(scale <q, k>) divided
by its own sum, for heads of channels, and neither K nor the normalised weights are ever stored.  The gradient stands beside it
as `cdist_grad` stands beside `cdist`.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _native
from .build_a_kernel import _call_result, _current_stream_for, _is_cuda, _torch_call_for

__all__ = ["cross_attention", "cross_attention_grad", "prefix_attention"]

_MAX_EXTENT = 0x7fffffff      # of the 32-bit fields of KmAttentionArgs
_TYPES = {torch.float32: _native.TYPE_FLOAT32, torch.bfloat16: _native.TYPE_BFLOAT16, torch.float16: _native.TYPE_FLOAT16}


def _check_operand(name, t, like, dims):
    """A CUDA tensor of the type and device of `like` with contiguous channels and one of `dims` numbers of dimensions."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a PyTorch tensor")
    if t.dtype != like.dtype or t.dtype not in _TYPES:
        raise TypeError(f"{name} must have dtype torch.float32, torch.bfloat16 or torch.float16, the same as q: got {t.dtype}")
    if not _is_cuda(t):
        raise ValueError(f"{name} must be on a CUDA device")
    if t.device != like.device:
        raise ValueError("All inputs must be on the same CUDA device")
    if t.dim() not in dims:
        raise ValueError(f"{name} must have {' or '.join(map(str, dims))} dimensions, got {t.dim()}")
    if t.size(-1) > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have stride 1 in last dimension")
    if max(t.shape) > _MAX_EXTENT:
        raise ValueError(f"the extents of {name} must be below 2^31, got {tuple(t.shape)}")


def _batch(name: str, L: int, t: torch.Tensor) -> int:
    batch = t.size(0) if t.dim() == 4 else 1
    if batch != 1 and L != 1 and batch != L:
        raise ValueError(f"{name} batch size of {batch} does not match with another non-one batch size, {L}")
    return batch if L == 1 else L


def _heads(t: Optional[torch.Tensor]) -> _native.KmHeads:
    """A (rows, heads, channels) or (batch, rows, heads, channels) tensor; a batch of one broadcasts."""
    if t is None:
        return _native.KmHeads()
    stride_l = t.stride(0) if t.dim() == 4 and t.size(0) != 1 else 0
    return _native.KmHeads(t.data_ptr(), stride_l, t.stride(-3), t.stride(-2))


def _check_written(name, t, like, shape):
    _check_operand(name, t, like, (4,))
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_lse(name, lse, q, L, H, N):
    if not isinstance(lse, torch.Tensor):
        raise TypeError(f"{name} must be a PyTorch tensor")
    if lse.dtype != torch.float32:
        raise TypeError(f"{name} must have dtype torch.float32")
    if not _is_cuda(lse) or lse.device != q.device:
        raise ValueError(f"{name} must be on the same CUDA device as inputs")
    if tuple(lse.shape) != (L, H, N):
        raise ValueError(f"{name} must have shape (L={L}, H={H}, N={N}), got {tuple(lse.shape)}")
    if N > 1 and lse.stride(-1) != 1:
        raise ValueError(f"{name} must have stride 1 in last dimension")


def _marshal(q, k, v, lengths, scale, prefix=None):
    """Checks what the three operators share; (KmAttentionArgs with the inputs filled in, L)."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a PyTorch tensor")
    for name, t in (('q', q), ('k', k), ('v', v)):
        _check_operand(name, t, q, (3, 4))
    N, H, D = q.shape[-3:]
    M, Hk, D_k = k.shape[-3:]
    if D_k != D:
        raise ValueError(f"q and k must have the same number of channels: got {D} and {D_k}")
    if D < 1 or D > 256:
        raise ValueError(f"the number of channels must be in [1, 256], got {D}")
    if tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"v must have the shape of k, {tuple(k.shape)}, got {tuple(v.shape)}")
    if Hk < 1 or H % Hk != 0:
        raise ValueError(f"the heads of q ({H}) must be a multiple of those of k ({Hk})")
    L = 1
    for name, t in (('q', q), ('k', k), ('v', v)):
        L = _batch(name, L, t)
    if L > 1 and M > 0 and (_heads(k).stride_l == 0) != (_heads(v).stride_l == 0):
        raise ValueError("k and v must both be broadcast over the batch, or neither")
    args = _native.KmAttentionArgs()
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor):
            raise TypeError("lengths must be a PyTorch tensor if provided")
        if lengths.dtype != torch.int32:
            raise TypeError("lengths must have dtype torch.int32")
        if not _is_cuda(lengths) or lengths.device != q.device:
            raise ValueError("lengths must be on the same CUDA device as inputs")
        if lengths.dim() != 1 or (lengths.size(0) != L and L != 1):
            raise ValueError(f"lengths must have shape (L={L},), got {tuple(lengths.shape)}")
        if lengths.size(0) > _MAX_EXTENT:
            raise ValueError(f"the extents of lengths must be below 2^31, got {tuple(lengths.shape)}")
        L = lengths.size(0)
        args.lengths, args.lengths_stride = lengths.data_ptr(), lengths.stride(0) if L > 1 else 0
    if prefix is not None:
        for name, t in zip(('k_prefix', 'v_prefix'), prefix):
            _check_operand(name, t, q, (3,))
            if tuple(t.shape[-2:]) != (Hk, D):
                raise ValueError(f"{name} must have shape (P, {Hk}, {D}), got {tuple(t.shape)}")
        if prefix[0].shape != prefix[1].shape:
            raise ValueError(f"v_prefix must have the shape of k_prefix, {tuple(prefix[0].shape)}, got {tuple(prefix[1].shape)}")
        args.prefix = prefix[0].size(0)
        args.k_prefix, args.v_prefix = _heads(prefix[0]), _heads(prefix[1])
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    scale = float(scale)
    if not (math.isfinite(scale) and scale >= 0.0):
        raise ValueError(f"scale must be finite and not negative, got {scale}")
    args.l, args.n, args.m, args.heads, args.key_heads, args.d = L, N, M, H, Hk, D
    args.type, args.scale = _TYPES[q.dtype], scale
    args.q, args.k, args.v = _heads(q), _heads(k), _heads(v)
    return args, L


def _launch(args, kind, q, debug):
    stream_ptr = _current_stream_for(q.device)
    need = _native.attention_scratch_bytes(args, kind)
    scratch = None
    if need > 0:
        try:
            scratch = torch.empty(need // 4, dtype=torch.float32, device=q.device)
            args.scratch, args.scratch_bytes = scratch.data_ptr(), need
        except torch.cuda.OutOfMemoryError:      # there it only makes the call faster
            if kind != _native.ATTENTION_CROSS:
                raise
    if debug:
        print(f'(Kermac Debug) Launching kernel: {_native.describe_attention(args, kind)}')
    _native.launch_attention(args, kind, stream_ptr)


def _forward(kind, q, k, v, lengths, scale, out, lse, return_lse, debug, prefix=None):
    # An ordinary call goes straight to the C-ABI (csrc/km_torch_call.cpp); what that declines (None) is checked below.
    call = _native._call
    if call is None:
        call = _torch_call_for(q)
    if call and not debug:
        result = call.attention(kind, q, k, v, *(prefix or (None, None)), lengths, scale, out, lse, return_lse)
        if result is not None:
            return _call_result(result, _native.ATTENTION_SYMBOLS[kind])
    args, L = _marshal(q, k, v, lengths, scale, prefix)
    N, H, D = q.shape[-3:]
    if out is None:
        out = torch.empty((L, N, H, D), dtype=q.dtype, device=q.device)
    else:
        _check_written('out', out, q, (L, N, H, D))
    if lse is not None:
        _check_lse('lse', lse, q, L, H, N)
    elif return_lse:
        lse = torch.empty((L, H, N), dtype=torch.float32, device=q.device)
    args.out = _heads(out)
    if lse is not None:
        args.lse, args.lse_stride_l, args.lse_stride_head = lse.data_ptr(), lse.stride(0), lse.stride(1)
    _launch(args, kind, q, debug)
    return (out, lse) if return_lse else out


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    debug=False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """out[l, n, h] = sum_m softmax_m(scale * <q[l, n, h], k[l, m, h']>) * v[l, m, h'],  h' = h // (H / Hk).

    q: (N, H, D) or (L, N, H, D) queries; k, v: (M, Hk, D) or (L, M, Hk, D), the states they look at; float32, bfloat16 or
    float16 CUDA tensors of one type, any strides but the last, which is 1 (heads held first are passed as
    `x.transpose(-3, -2)`).  H is a multiple of Hk, 1 <= D <= 256.  Batch extents must be 1 or agree; extent-1 operands
    broadcast, and k and v that the whole batch shares are read once for all.  `lengths`: (L,) int32 on the device, how many of
    the M states each batch entry has (None: all; values outside [0, M] count as the nearest of the two); what lies
    behind is never used, whatever it holds.  A query without a state to look at gets zeros and lse = -inf.

    `out`: (L, N, H, D), allocated when None.  `lse`: (L, H, N) float32 for the logarithm of each query's sum of exponentials, which
    `cross_attention_grad` needs; with `return_lse` the call returns (out, lse).  Neither may share memory with an input.  `scale` is
    1 / sqrt(D) when None.

    Scores, softmax and sums are 32-bit; with 16-bit types the weights are rounded to that type for the product with v.  float32 inputs
    are taken apart into three bfloat16 or two tf32 parts: those that are used have to be finite and below 2^127.  Equal calls give
    equal bits.  Partial sums, where few queries look at many states (at most 512 MB), and copies of float32 inputs
    of up to 64 channels (384 bytes a row of a head, at most 1 GiB) are taken from torch's allocator for the duration of the call.
    Launches on torch's current stream and returns without synchronising; like every allocation by torch that has to be
    captured through torch.cuda.graph.

    Bounded waits as in `kernel_matvec`: one that runs out leaves rows unwritten and raises the flag that
    `kermac_b200._native.device_error_flag()` reads.
    """
    return _forward(_native.ATTENTION_CROSS, q, k, v, lengths, scale, out, lse, return_lse, debug)


def prefix_attention(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    debug=False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the N newest tokens of each of L sequences that continue one shared prefix.

    q: (L, N, H, D); k_prefix, v_prefix: (P, Hk, D), the prefix, read and multiplied once for the whole batch; k, v: (L, M, Hk, D),
    each sequence's own tokens, of which `lengths` (or all M) are there, the N newest included.  Query n sees the whole prefix
    and own token j when j <= lengths[l] - N + n; a v that is not finite reaches, as 0 * inf, the queries before it too.  P and M may be 0.  Everything else as in `cross_attention`, but for the partial sums: where
    there are both a prefix and own tokens each of the two takes 4 (D + 2) bytes a query and head at least, without a limit.
    """
    return _forward(_native.ATTENTION_PREFIX, q, k, v, lengths, scale, out, lse, return_lse, debug, prefix=(k_prefix, v_prefix))


def cross_attention_grad(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    grad_out: torch.Tensor,
    lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    grad_q: Optional[torch.Tensor] = None,
    grad_k: Optional[torch.Tensor] = None,
    grad_v: Optional[torch.Tensor] = None,
    debug=False,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(grad_q, grad_k, grad_v) of `cross_attention` for the gradient grad_out of its result.

    `out` (L, N, H, D) and `lse` (L, H, N) are what cross_attention(..., return_lse=True) returned for the same q, k, v, lengths and
    scale; grad_out has the shape of out.  Each gradient has its input's shape with a batch dimension: an input that was broadcast
    over the batch (extent 1) gets the sum over the batch, key heads that several query heads share the sum over these, and
    states behind `lengths` get zeros.  grad_q, grad_k, grad_v: destinations of those shapes, which share memory with nothing else that
    the call is given, allocated when None.

    Sums are 32-bit and in a fixed order: equal calls give equal bits.  Weights are taken from `lse`, whose rounding to float32 is a
    factor on all of a row's: 3 % where scores are of size 10^6.  Takes scratch from torch's allocator for the duration
    of the call: 4 bytes a query and head (float16: some more), another 4 D where q is broadcast over the batch, and partial sums where
    sums over states or queries are divided (at most 256 MB for each gradient).
    """
    call = _native._call
    if call is None:
        call = _torch_call_for(q)
    if call and not debug and grad_q is None and grad_k is None and grad_v is None:
        result = call.attention_grad(q, k, v, out, lse, grad_out, lengths, scale)
        if result is not None:
            return _call_result(result, _native.ATTENTION_SYMBOLS[_native.ATTENTION_GRAD])
    args, L = _marshal(q, k, v, lengths, scale)
    N, H, D = q.shape[-3:]
    M, Hk = k.shape[-3:-1]
    for name, t in (('out', out), ('grad_out', grad_out)):
        _check_operand(name, t, q, (4,))
        if tuple(t.shape) != (L, N, H, D):
            raise ValueError(f"{name} must have shape {(L, N, H, D)}, got {tuple(t.shape)}")
    _check_lse('lse', lse, q, L, H, N)
    args.q_batch = q.size(0) if q.dim() == 4 else 1
    args.kv_batch = k.size(0) if k.dim() == 4 else 1
    if (v.size(0) if v.dim() == 4 else 1) != args.kv_batch:
        raise ValueError("k and v must have the same batch size")
    grads = []
    for name, t, shape in (('grad_q', grad_q, (args.q_batch, N, H, D)), ('grad_k', grad_k, (args.kv_batch, M, Hk, D)),
                           ('grad_v', grad_v, (args.kv_batch, M, Hk, D))):
        if t is None:
            t = torch.empty(shape, dtype=q.dtype, device=q.device)
        else:
            _check_written(name, t, q, shape)
        grads.append(t)
    args.out, args.grad_out = _heads(out), _heads(grad_out)
    args.grad_q, args.grad_k, args.grad_v = map(_heads, grads)
    args.lse, args.lse_stride_l, args.lse_stride_head = lse.data_ptr(), lse.stride(0), lse.stride(1)
    _launch(args, _native.ATTENTION_GRAD, q, debug)
    return tuple(grads)
