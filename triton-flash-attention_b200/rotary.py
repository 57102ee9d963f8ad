"""Queries and keys on their way into the attention: a root-mean-square norm
of every head and the rotation by the token's position, in one pass.

No counterpart in the reference, whose API takes queries and keys as they
enter the product (triton_flash_attention/attention.py:584-626).  For a row
``x`` of ``D`` values (one head of one token)::

    y = x / sqrt(mean(x^2) + eps) * weight
    y'[a] = y[a] cos - y[b] sin,   y'[b] = y[b] cos + y[a] sin

for the column pairs ``(a, b)`` of the first ``rotary_dim`` columns; columns
behind them keep ``y``.  Both steps run in fp32 and the result is rounded
once (bf16 rows whose squares leave fp32's range are scaled first).
``qk_norm_rotary`` supports autograd; ``paged_append`` (``paging.py``) is the
same preparation for serving, with keys and values written to a paged cache.
"""

from __future__ import annotations

import math
from numbers import Real

import torch

from . import _abi
from .attention import SUPPORTED_DTYPES, SUPPORTED_HEAD_DIMS, _device_capability

# rows of the partial weight gradients (FA_ROTARY_PARTIALS of include/fa_b200.h)
ROTARY_PARTIALS = 592


def rotary_table(max_positions: int, rotary_dim: int, *, base: float = 10000.0, device=None) -> torch.Tensor:
    """The ``(max_positions, rotary_dim)`` fp32 table that the rotating calls
    take: for each position the ``rotary_dim / 2`` cosines, then the sines, of
    ``position * base ** (-2 i / rotary_dim)``, from 64-bit angles (far
    positions need them).  Made once and kept; any other frequencies can be
    put in a table of the same layout."""
    for name, v in (("max_positions", max_positions), ("rotary_dim", rotary_dim)):
        if isinstance(v, bool) or not isinstance(v, int) or v <= 0:
            raise ValueError(f"{name} must be a positive int")
    if rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16")
    if isinstance(base, bool) or not isinstance(base, Real) or not math.isfinite(base) or base <= 0:
        raise ValueError("base must be a finite positive number")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def check_backend(tensor: torch.Tensor) -> None:
    """Raises unless the B200 kernels serve tensors of this device, type and
    head dim, with the messages of the attention calls."""
    if not tensor.is_cuda:
        raise RuntimeError("B200 CUDA backend is unavailable: the B200 kernel requires a CUDA tensor")
    if tensor.dtype not in SUPPORTED_DTYPES:
        raise RuntimeError("B200 CUDA backend is unavailable: the custom mixed-precision path currently "
                           "supports float16 and bfloat16")
    if tensor.shape[-1] not in SUPPORTED_HEAD_DIMS:
        supported = ", ".join(str(dim) for dim in SUPPORTED_HEAD_DIMS)
        raise RuntimeError(f"B200 CUDA backend is unavailable: head_dim must be one of ({supported}) "
                           "for the B200 path")
    if _device_capability(tensor.device) != (10, 0):
        raise RuntimeError("B200 CUDA backend is unavailable: the kernels are built for sm_100a (B200) GPUs only")


def launch(tensor: torch.Tensor, what: str, dtype, *args) -> None:
    """Calls the entry ``what`` for operands of ``dtype`` (None: the entry has
    no type) with ``args`` and the tensor's device's current stream, on that
    device.  (Calls of a few microseconds of GPU time are bound by their host
    side: this asks for no more than it has to.)"""
    fn, pack = _abi.packed_entry(what, dtype)
    index = tensor.get_device()
    if torch._C._cuda_getDevice() == index:
        rc = fn(pack(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            rc = fn(pack(*args, torch._C._cuda_getCurrentRawStream(index)))
    if rc:
        _abi.check(rc, what)


_UNSEEN = object()
_row_strides: dict = {}


def _strides_arg(s: tuple):
    """{batch, head, seq} strides of a (B, H, N, D) or packed (total, H, D)
    tensor for the library, or None when its rows cannot be read 16 bytes at a
    time: unit stride over D, the others multiples of 8 elements.  A packed
    tensor has one batch, whose stride is of no consequence."""
    if s[-1] != 1 or any(x % 8 for x in s[:-1]):
        return None
    return _abi.strides_of(s[:3] if len(s) == 4 else (8, s[1], s[0]))


def row_arg(t: torch.Tensor):
    """``(tensor, address, strides)`` of rows to be read 16 bytes at a time:
    ``t`` itself where its strides and start allow it, else a copy."""
    s = t.stride()
    arr = _row_strides.get(s, _UNSEEN)
    if arr is _UNSEEN:
        if len(_row_strides) > 1024:
            _row_strides.clear()
        arr = _row_strides[s] = _strides_arg(s)
    p = t.data_ptr()
    if arr is not None and not p & 15:
        return t, p, arr
    return row_arg(torch.empty(t.shape, device=t.device, dtype=t.dtype).copy_(t))


def check_table(table, rotary_max: int, device) -> None:
    if not isinstance(table, torch.Tensor):
        raise TypeError("table must be a torch.Tensor")
    shape = table.shape
    if len(shape) != 2 or table.dtype != torch.float32 or not table.is_contiguous() or shape[0] == 0:
        raise ValueError("table must be a contiguous (max_positions, rotary_dim) float32 tensor")
    rd = shape[1]
    if rd == 0 or rd % 16 or rd > rotary_max:
        raise ValueError(f"the table's rotary_dim must be a multiple of 16 up to the head dim {rotary_max}; got {rd}")
    if table.device != device:
        raise ValueError("table must be on the same device as query")
    if table.data_ptr() % 16:
        raise ValueError("table must start on a 16-byte boundary")


def check_weights(query_weight, key_weight, query) -> None:
    if (query_weight is None) != (key_weight is None):
        raise ValueError("pass both query_weight and key_weight, or neither for the rotation alone")
    if query_weight is None:
        return
    d, device = query.shape[-1], query.device
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if w.shape != (d,) or w.device != device:
            raise ValueError(f"{name} must be a 1-D tensor of head_dim weights on the query's device")
    dtype = query_weight.dtype
    if dtype != torch.float32 and dtype != query.dtype:
        raise ValueError("query_weight and key_weight must have the query's dtype or float32")
    if dtype != key_weight.dtype:
        raise ValueError("query_weight and key_weight must have the same dtype")


def check_eps(eps) -> None:
    if type(eps) is float and 0.0 <= eps < math.inf:
        return
    if isinstance(eps, bool) or not isinstance(eps, Real) or not 0.0 <= eps < math.inf:
        raise ValueError("eps must be a finite non-negative number")


def _validate(query, key, table, positions, query_weight, key_weight, eps, interleaved) -> None:
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    if not isinstance(key, torch.Tensor):
        raise TypeError("key must be a torch.Tensor")
    qs, ks, ndim, dev = query.shape, key.shape, query.ndim, query.device
    for name, shape in (("query", qs), ("key", ks)):
        if len(shape) not in (3, 4):
            raise ValueError(f"{name} must have shape (batch, heads, sequence, head_dim) or (total, heads, head_dim); "
                             f"got {tuple(shape)}")
        if 0 in shape:
            raise ValueError(f"{name} dimensions must all be greater than zero")
    if ndim != len(ks):
        raise ValueError("query and key must have the same layout")
    if dev != key.device:
        raise ValueError("query and key must be on the same device")
    if query.dtype != key.dtype:
        raise ValueError("query and key must have the same dtype")
    if qs[-1] != ks[-1]:
        raise ValueError("query and key head dimensions must match")
    if ndim == 4:
        n = qs[2]
        if qs[0] != ks[0] or n != ks[2]:
            raise ValueError("query and key batch and sequence dimensions must match")
    else:
        n = qs[0]
        if n != ks[0]:
            raise ValueError("query and key must have the same number of rows")
    if not isinstance(interleaved, bool):
        raise TypeError("interleaved must be a bool")
    check_eps(eps)
    check_table(table, qs[-1], dev)
    check_weights(query_weight, key_weight, query)
    if positions is None:
        if ndim == 3:
            raise ValueError("packed (total, heads, head_dim) tensors need positions")
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be a torch.Tensor")
        ps = positions.shape
        fits = (len(ps) == 1 and ps[0] == n) or (ndim == 4 and len(ps) == 2 and ps[0] == qs[0] and ps[1] == n)
        if not fits or positions.dtype != torch.int32 or positions.device != dev:
            raise ValueError("positions must be an int32 tensor of the token dimension, or of (batch, sequence) for "
                             "4-D tensors, on the query's device")
    check_backend(query)


def _sizes(q, k):
    """(B, Hq, Hkv, N, D)"""
    s = q.shape
    if len(s) == 4:
        return s[0], s[1], k.shape[1], s[2], s[3]
    return 1, s[1], k.shape[1], s[0], s[2]


def _contiguous_strides(shape):
    """Strides of an output of that shape: contiguous."""
    *_, h, n, d = shape
    return _strides_arg((h * n * d, n * d, d, 1) if len(shape) == 4 else (n * d, d, 1))


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _contiguous_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(q, k, table, positions, query_weight, key_weight, eps, interleaved):
    """The forward's launch; besides the outputs what the backward's takes of
    it: the rows as they were read, the sizes, and the arguments both have of the
    outputs' and of positions."""
    q, qp, qs = row_arg(q)
    k, kp, ks = row_arg(k)
    b, hq, hkv, n, d = _sizes(q, k)
    max_positions, rd = table.shape
    fp32 = query_weight is not None and query_weight.dtype == torch.float32
    per_batch = n if positions is not None and positions.ndim == 2 else 0
    qo, ko = _contiguous_like(q), _contiguous_like(k)
    _, qop, qos = row_arg(qo)
    _, kop, kos = row_arg(ko)
    launch(q, "fa_qk_norm_rotary", q.dtype, qp, kp, qop, kop, table.data_ptr(), _ptr(positions), _ptr(query_weight),
           _ptr(key_weight), b, hq, hkv, n, d, max_positions, rd, interleaved, fp32, qs.at, ks.at, qos.at,
           kos.at, per_batch, eps)
    return qo, ko, q, k, (b, hq, hkv, n, d, max_positions, rd, interleaved, fp32), (qos, kos, per_batch, eps)


def _backward(q, k, grad_q, grad_k, table, positions, query_weight, key_weight, sizes, rest, weight_grads):
    """The backward's launch, with ``sizes`` and ``rest`` of ``_forward``.  (It
    runs on autograd's own thread, where host work costs more: what the
    forward worked out is not worked out again.  The rows' strides are: a hook
    on saved tensors may give them back laid out otherwise.)"""
    q, qp, qs = row_arg(q)
    k, kp, ks = row_arg(k)
    grad_q, gqp, gqs = row_arg(grad_q)
    grad_k, gkp, gks = row_arg(grad_k)
    qos, kos, per_batch, eps = rest
    dq, dk = _contiguous_like(q), _contiguous_like(k)
    dwq = dwk = part = None
    if weight_grads:
        dwq, dwk = torch.empty_like(query_weight), torch.empty_like(key_weight)
        part = table.new_empty(ROTARY_PARTIALS * sizes[4])
    launch(q, "fa_qk_norm_rotary_bwd", q.dtype, qp, kp, gqp, gkp, dq.data_ptr(), dk.data_ptr(),
           _ptr(dwq), _ptr(dwk), _ptr(part), table.data_ptr(), _ptr(positions), _ptr(query_weight), _ptr(key_weight),
           *sizes, qs.at, ks.at, gqs.at, gks.at, qos.at, kos.at, per_batch, eps)
    return dq, dk, dwq, dwk


def _contiguous(*tensors):
    return [None if t is None else t.contiguous() for t in tensors]


def qk_norm_rotary_forward(q, k, table, positions, query_weight, key_weight, eps: float, interleaved: bool):
    """Launch the forward: contiguous outputs in the inputs' layout."""
    _validate(q, k, table, positions, query_weight, key_weight, eps, interleaved)
    positions, query_weight, key_weight = _contiguous(positions, query_weight, key_weight)
    return _forward(q, k, table, positions, query_weight, key_weight, eps, interleaved)[:2]


def qk_norm_rotary_backward(q, k, grad_q, grad_k, table, positions, query_weight, key_weight, eps: float,
                            interleaved: bool, weight_grads: bool = True):
    """dQ, dK and, with weights and ``weight_grads``, the weights' gradients
    (else None).  Gradients repeat bit for bit."""
    for name, g, t in (("grad_q", grad_q, q), ("grad_k", grad_k, k)):
        if not isinstance(g, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if isinstance(t, torch.Tensor) and (g.shape != t.shape or g.dtype != t.dtype or g.device != t.device):
            raise ValueError(f"{name} must have the shape, dtype and device of its output")
    _validate(q, k, table, positions, query_weight, key_weight, eps, interleaved)
    positions, query_weight, key_weight = _contiguous(positions, query_weight, key_weight)
    qos, kos = _contiguous_strides(q.shape), _contiguous_strides(k.shape)
    sizes = (*_sizes(q, k), *table.shape, interleaved,
             query_weight is not None and query_weight.dtype == torch.float32)
    per_batch = sizes[3] if positions is not None and positions.ndim == 2 else 0
    return _backward(q, k, grad_q, grad_k, table, positions, query_weight, key_weight, sizes,
                     (qos, kos, per_batch, eps), weight_grads and query_weight is not None)


class B200QKNormRotary(torch.autograd.Function):
    """Autograd bridge; saves the inputs only (a row's norm is found again
    from its values, which the backward reads anyhow)."""

    @staticmethod
    def forward(ctx, query, key, table, positions, query_weight, key_weight, eps, interleaved):
        qo, ko, query, key, ctx.sizes, ctx.rest = _forward(query, key, table, positions, query_weight, key_weight, eps,
                                                           interleaved)
        ctx.save_for_backward(query, key, table, positions, query_weight, key_weight)
        return qo, ko

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        if torch.is_grad_enabled():
            raise RuntimeError("qk_norm_rotary is differentiable once: its backward has no gradient (create_graph)")
        query, key, table, positions, query_weight, key_weight = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dq, dk, dwq, dwk = _backward(query, key, grad_query, grad_key, table, positions, query_weight, key_weight,
                                     ctx.sizes, ctx.rest, needs[4] or needs[5])
        return dq, dk, None, None, dwq, dwk, None, None


def qk_norm_rotary(query, key, table, positions=None, *, query_weight=None, key_weight=None, eps: float = 1e-6,
                   interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm and rotate queries and keys for the attention calls.

    ``query``, ``key``: ``(B, Hq, N, D)`` and ``(B, Hkv, N, D)``, or packed
    ``(total, Hq, D)`` and ``(total, Hkv, D)``; views of a fused projection
    are read in place.  ``table``: ``rotary_table``'s; its width is the number
    of columns that turn.  ``positions``: int32, ``(N,)`` or ``(B, N)``, or
    ``(total,)`` when packed; None counts from 0 (4-D only).  ``query_weight``,
    ``key_weight``: ``D`` weights each, in the operand type or float32; with
    both None there is no norm.  ``interleaved`` pairs columns ``(2 i, 2 i +
    1)`` instead of ``(i, i + rotary_dim / 2)``.  Returns contiguous tensors
    in the inputs' layout and supports autograd for the queries, keys and
    weights.

    A position outside the table is found on the GPU: its turned columns are
    NaN and the device status (``_abi.device_status``) names the error."""
    _validate(query, key, table, positions, query_weight, key_weight, eps, interleaved)
    positions, query_weight, key_weight = _contiguous(positions, query_weight, key_weight)
    return B200QKNormRotary.apply(query, key, table, positions, query_weight, key_weight, float(eps), interleaved)
