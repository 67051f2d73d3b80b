"""Learned relative position bias by buckets, with the gradient of its table.

Position pairs are sorted into buckets by their distance, and every bucket has a learned row.  The
pair stack of a structure model starts from it (``pair[b,i,j,:] += table[bucket(i, j), :]``), and an
attention adds one column of it per head to its scores (``bias[h,i,j] = table[bucket(i, j), h]``);
``cross_attention_b200`` takes that form as its ``bias``.  Forward and gradient are single passes over
the large tensor through the C-ABI library.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch
import torch.nn as nn

from . import _lib
from .functional import _dtype_code, _on_device, _require_cuda, _require_no_tangent, _stream_handle

__all__ = ["PositionBuckets", "relative_position_bias_b200", "relative_position_bias_backward_b200",
           "RelativePositionBiasB200"]

_LAYOUTS = {"heads": _lib.RELPOS_HEADS, "pair": _lib.RELPOS_PAIR}


class PositionBuckets:
    """Rule that sorts a pair of positions into a bucket by ``d = q_pos - k_pos``.

    ``clipped(r)``: ``clip(d, -r, r) + r``, i.e. ``2 r + 1`` buckets.  ``logarithmic(n, top)``: ``n / 2``
    buckets for ``d >= 0`` followed by as many for ``d < 0``; distances below ``n / 4`` have a bucket
    each, longer ones share buckets evenly spaced in the logarithm up to ``top``, beyond which there
    is one; with ``bidirectional=False`` all ``n`` buckets are for ``max(d, 0)``.  The borders of the
    logarithmic buckets are whole numbers found in exact arithmetic: bucket ``near + k`` starts at the
    smallest ``t`` with ``(t / near)^(m) >= (top / near)^k``, ``m`` the number of shared buckets.
    ``segments=True`` adds a last bucket for pairs of different segments (chains).  ``rows`` is the
    number of rows a table needs."""

    def __init__(self, kind: int, count: int, max_distance: int, thresholds: tuple, segments: bool):
        self.kind, self.count, self.max_distance, self.segments = kind, count, max_distance, bool(segments)
        self.thresholds = thresholds
        self.rows = count + self.segments
        if self.rows > _lib.MAX_BUCKETS:
            raise NotImplementedError(f"at most {_lib.MAX_BUCKETS} buckets are supported, got {self.rows}")
        if (thresholds[-1] if thresholds else max_distance) > _lib.MAX_LUT:
            raise NotImplementedError(f"distances beyond {_lib.MAX_LUT} must share a bucket")
        if len(thresholds) > _lib.MAX_THRESHOLDS:
            raise NotImplementedError(f"at most {_lib.MAX_THRESHOLDS} shared buckets a side are supported, got {len(thresholds)}")
        self._struct = _lib.Buckets(kind, count, max_distance, int(self.segments), len(thresholds),
                                    (C.c_int32 * _lib.MAX_THRESHOLDS)(*thresholds))

    @property
    def _address(self) -> int:
        """Where the library reads the rule; asked for at every call, since a copy (``copy.deepcopy``, pickle) has a
        structure of its own."""
        return C.addressof(self._struct)

    @staticmethod
    @functools.lru_cache(maxsize=256)
    def clipped(max_distance: int, *, segments: bool = False) -> "PositionBuckets":
        if max_distance < 0:
            raise ValueError(f"max_distance must not be negative, got {max_distance}")
        return PositionBuckets(_lib.BUCKETS_CLIPPED, 2 * max_distance + 1, max_distance, (), segments)

    @staticmethod
    @functools.lru_cache(maxsize=256)
    def logarithmic(num_buckets: int, max_distance: int, *, bidirectional: bool = True,
                    segments: bool = False) -> "PositionBuckets":
        if bidirectional and num_buckets % 2:
            raise ValueError(f"num_buckets must be even for two directions, got {num_buckets}")
        side = num_buckets // 2 if bidirectional else num_buckets
        near = side // 2
        if near < 1:
            raise ValueError(f"num_buckets = {num_buckets} leaves no bucket for near distances")
        if max_distance <= near:
            raise ValueError(f"max_distance must be more than the {near} near distances, got {max_distance}")
        if num_buckets > _lib.MAX_BUCKETS:
            raise NotImplementedError(f"at most {_lib.MAX_BUCKETS} buckets are supported, got {num_buckets}")
        shared, thresholds, t = side - near, [], near
        for k in range(1, shared):
            want = near ** (shared - k) * max_distance ** k
            while t ** shared < want:
                t += 1
                if t > _lib.MAX_LUT:
                    raise NotImplementedError(f"distances beyond {_lib.MAX_LUT} must share a bucket")
            thresholds.append(t)
        kind = _lib.BUCKETS_LOG if bidirectional else _lib.BUCKETS_CAUSAL
        return PositionBuckets(kind, num_buckets, max_distance, tuple(thresholds), segments)

    def __repr__(self) -> str:
        name = ("clipped", "logarithmic", "logarithmic one-sided")[self.kind]
        return f"PositionBuckets({name}, rows={self.rows}, max_distance={self.max_distance}, segments={self.segments})"


def _index(t, name: str, device):
    """``(tensor, wide, batch or None, batch stride)`` of a position or segment vector."""
    if t.dtype is torch.int32:
        wide = 0
    elif t.dtype is torch.int64:
        wide = 1
    else:
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dim() not in (1, 2):
        raise ValueError(f"{name} must be [L] or [B, L], got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    if t.dim() == 1:
        return t, wide, None, 0
    return t, wide, t.shape[0], t.stride(0) if t.shape[0] > 1 else 0


class _Call:
    """Checked positions of one call and the descriptor they give."""

    def __init__(self, buckets, q_pos, k_pos, q_segment, k_segment, layout, dtype_code, table_code, channels, device):
        if not isinstance(buckets, PositionBuckets):
            raise ValueError("buckets must be a PositionBuckets")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be heads|pair, got {layout!r}")
        if k_pos is None:
            k_pos = q_pos
        if buckets.segments:
            if q_segment is None:
                raise ValueError("these buckets tell segments apart: q_segment is needed")
            if k_segment is None:
                if k_pos is not q_pos:
                    raise ValueError("k_pos without k_segment")
                k_segment = q_segment
        elif q_segment is not None or k_segment is not None:
            raise ValueError("segments were given, but the buckets do not tell them apart")
        qp, w0, b0, s0 = _index(q_pos, "q_pos", device)
        kp, w1, b1, s1 = (qp, w0, b0, s0) if k_pos is q_pos else _index(k_pos, "k_pos", device)
        batches = {b0, b1}
        self.keep = [qp, kp]
        self.args = [qp.data_ptr(), kp.data_ptr(), None, None]
        wide, s2, s3 = w0 | w1 << 1, 0, 0
        if buckets.segments:
            qs, w2, b2, s2 = _index(q_segment, "q_segment", device)
            ks, w3, b3, s3 = (qs, w2, b2, s2) if k_segment is q_segment else _index(k_segment, "k_segment", device)
            if qs.shape[-1] != qp.shape[-1] or ks.shape[-1] != kp.shape[-1]:
                raise ValueError("segments must have the length of their positions")
            batches |= {b2, b3}
            self.keep += [qs, ks]
            self.args[2:] = [qs.data_ptr(), ks.data_ptr()]
            wide |= w2 << 2 | w3 << 3
        batches.discard(None)
        if len(batches) > 1:
            raise ValueError(f"positions and segments have different batch sizes: {sorted(batches)}")
        self.batch = batches.pop() if batches else None
        self.lq, self.lk, self.channels = qp.shape[-1], kp.shape[-1], channels
        B = 1 if self.batch is None else self.batch
        self.empty = B == 0 or self.lq == 0 or self.lk == 0 or channels == 0
        self.head = (_lib.RELPOS_DESC.size, _LAYOUTS[layout], dtype_code, table_code, B, self.lq, self.lk, channels, wide, 0,
                     s0, s1, s2, s3)

    def shape(self, layout):
        lead = () if self.batch is None else (self.batch,)
        return (*lead, self.channels, self.lq, self.lk) if layout == "heads" else (*lead, self.lq, self.lk, self.channels)

    def pack(self, t=None) -> bytes:
        """``trimul_relpos_desc``, with the strides of the heads tensor ``t``."""
        if t is None:
            return _lib.RELPOS_DESC.pack(*self.head, 0, 0, 0)
        strides = t.stride()
        return _lib.RELPOS_DESC.pack(*self.head, strides[0] if self.batch is not None else 0, strides[-3], strides[-2])


_workspace_sizes: dict = {}      # of the library's answers, by what they depend on


def _forward(table, buckets, q_pos, k_pos, q_segment, k_segment, layout, add, dtype):
    _require_cuda(table, "table")
    device = table.device
    if table.dim() != 2 or not isinstance(buckets, PositionBuckets) or table.shape[0] != buckets.rows:
        raise ValueError(f"table must be [{getattr(buckets, 'rows', 'buckets')}, channels], got {tuple(table.shape)}")
    if add is not None:
        if layout != "pair":
            raise ValueError("add is for the pair layout")
        if dtype is not None and dtype != add.dtype:
            raise ValueError(f"dtype {dtype} differs from that of add, {add.dtype}")
        if add.device != device:
            raise ValueError(f"add is on {add.device}, the table on {device}")
        dtype = add.dtype
    dtype = table.dtype if dtype is None else dtype
    code = _lib.dtype_code(dtype)
    call = _Call(buckets, q_pos, k_pos, q_segment, k_segment, layout, code, _dtype_code(table), table.shape[1], device)
    shape = call.shape(layout)
    if add is not None:
        if tuple(add.shape) != shape:
            raise ValueError(f"add must be {shape}, got {tuple(add.shape)}")
        add = add.detach() if add.requires_grad else add
        add = add if add.is_contiguous() else add.contiguous()
    table = table.detach() if table.requires_grad else table
    table = table if table.is_contiguous() else table.contiguous()
    with _on_device(device):
        if layout == "heads":
            # rows start on 16 bytes, which the kernels that read a bias rely on
            unit = 8 if code == _lib.DTYPE_BF16 else 4
            pitch = -(-call.lk // unit) * unit
            out = torch.empty(*shape[:-1], pitch, dtype=dtype, device=device)
            if pitch != call.lk:
                out = out[..., :call.lk]
            desc = call.pack(out)
        else:
            desc = call.pack()
            out = torch.empty(shape, dtype=dtype, device=device)
        if call.empty:
            return out
        rc = _lib.load().trimul_b200_relpos_bias(
            desc, buckets._address, table.data_ptr(), *call.args,
            add.data_ptr() if add is not None else None, out.data_ptr(), _stream_handle(device))
    _lib.check(rc, "trimul_b200_relpos_bias")
    return out


def relative_position_bias_backward_b200(grad: torch.Tensor, buckets: PositionBuckets, q_pos: torch.Tensor,
                                         k_pos: torch.Tensor | None = None, *, q_segment: torch.Tensor | None = None,
                                         k_segment: torch.Tensor | None = None, layout: str = "heads",
                                         dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Gradient of the table, ``[buckets.rows, channels]``, from the gradient of
    ``relative_position_bias_b200``'s result with the same positions: for each bucket the sum of
    ``grad`` over its position pairs.  Sums are held in fp32 and added in a fixed order (the same call
    gives the same bits), and rounded once to ``dtype``.  The gradient of ``add`` is ``grad`` itself."""
    _require_cuda(grad, "grad")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be heads|pair, got {layout!r}")
    if grad.dim() not in (3, 4):
        raise ValueError(f"grad must have three or four dimensions, got {tuple(grad.shape)}")
    device = grad.device
    channels = grad.shape[-3] if layout == "heads" else grad.shape[-1]
    call = _Call(buckets, q_pos, k_pos, q_segment, k_segment, layout, _dtype_code(grad), _lib.dtype_code(dtype), channels, device)
    if tuple(grad.shape) != call.shape(layout):
        raise ValueError(f"grad must be {call.shape(layout)}, got {tuple(grad.shape)}")
    grad = grad.detach() if grad.requires_grad else grad
    if layout == "pair":
        grad = grad if grad.is_contiguous() else grad.contiguous()
    else:
        if grad.shape[-1] > 1 and grad.stride(-1) != 1:
            grad = grad.contiguous()
    desc = call.pack(grad if layout == "heads" else None)
    with _on_device(device):
        out = torch.empty(buckets.rows, channels, dtype=dtype, device=device)
        if call.empty:
            return out.zero_()
        lib, key = _lib.load(), (call.head[:8], buckets)
        n = _workspace_sizes.get(key)
        if n is None:
            size = C.c_size_t()
            _lib.check(lib.trimul_b200_relpos_bias_grad_workspace_bytes(desc, buckets._address, C.byref(size)),
                       "trimul_b200_relpos_bias_grad_workspace_bytes")
            n = size.value
            if len(_workspace_sizes) >= 1024:
                _workspace_sizes.clear()
            _workspace_sizes[key] = n
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        rc = lib.trimul_b200_relpos_bias_grad(desc, buckets._address, *call.args, grad.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                              n, _stream_handle(device))
    _lib.check(rc, "trimul_b200_relpos_bias_grad")
    return out


class _RelativePositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, add, buckets, q_pos, k_pos, q_segment, k_segment, layout, dtype):
        # positions given twice are saved once: saved-tensor hooks may hand the backward pass two objects for them
        ctx.save_for_backward(q_pos, None if k_pos is q_pos else k_pos, q_segment, k_segment)
        ctx.buckets, ctx.layout, ctx.table_dtype = buckets, layout, table.dtype
        return _forward(table, buckets, q_pos, k_pos, q_segment, k_segment, layout, add, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q_pos, k_pos, q_segment, k_segment = ctx.saved_tensors
        dtable = None
        if ctx.needs_input_grad[0]:
            dtable = relative_position_bias_backward_b200(grad, ctx.buckets, q_pos, k_pos, q_segment=q_segment,
                                                          k_segment=k_segment, layout=ctx.layout, dtype=ctx.table_dtype)
        return dtable, grad if ctx.needs_input_grad[1] else None, None, None, None, None, None, None, None


def relative_position_bias_b200(table: torch.Tensor, buckets: PositionBuckets, q_pos: torch.Tensor,
                                k_pos: torch.Tensor | None = None, *, q_segment: torch.Tensor | None = None,
                                k_segment: torch.Tensor | None = None, layout: str = "heads",
                                add: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The rows of ``table`` that the position pairs' buckets select.

    ``table``: ``[buckets.rows, channels]``, bf16 or fp32.  ``q_pos``, ``k_pos`` (default: ``q_pos``):
    ``[Lq]``, ``[Lk]`` or with a leading batch axis, int32 or int64; values beyond ``2^30 - 1`` of either sign are
    taken as that value.  ``q_segment``, ``k_segment``: integers in the positions' shapes, for buckets with
    ``segments``; only their equality counts, so they may be any numbers.

    ``layout="heads"``: ``[(B,) channels, Lq, Lk]``, the form that ``cross_attention_b200`` takes as its
    bias.  Rows start on 16-byte boundaries: where ``Lk`` is not a multiple of 16 bytes, the result is a
    view into wider rows (and so not contiguous).  ``layout="pair"``: ``[(B,) Lq, Lk, channels]``, plus
    ``add`` where given (the pair tensor; the sum is rounded once).  The result has the dtype of
    ``add``, else ``dtype``, else that of the table.

    Differentiable in ``table`` and ``add`` in reverse mode; an input with a forward-mode tangent is refused.
    ``relative_position_bias_backward_b200`` is the gradient as a call of its own."""
    if torch.is_grad_enabled() and (table.requires_grad or (add is not None and add.requires_grad)):
        return _RelativePositionBias.apply(table, add, buckets, q_pos, k_pos, q_segment, k_segment, layout, dtype)
    _require_no_tangent("relative_position_bias_b200", table, add)
    return _forward(table, buckets, q_pos, k_pos, q_segment, k_segment, layout, add, dtype)


class RelativePositionBiasB200(nn.Module):
    """``relative_position_bias_b200`` with its table as a parameter (``weight``, ``[buckets.rows, channels]``).

    ``forward(q_pos, k_pos=None, q_segment=None, k_segment=None, add=None)``."""

    def __init__(self, buckets: PositionBuckets, channels: int, *, layout: str = "heads",
                 dtype: torch.dtype | None = None) -> None:
        super().__init__()
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be heads|pair, got {layout!r}")
        self.buckets, self.layout, self.dtype = buckets, layout, dtype
        self.weight = nn.Parameter(torch.empty(buckets.rows, channels))
        nn.init.normal_(self.weight, std=0.02)

    def forward(self, q_pos, k_pos=None, q_segment=None, k_segment=None, add=None):
        return relative_position_bias_b200(self.weight, self.buckets, q_pos, k_pos, q_segment=q_segment,
                                           k_segment=k_segment, layout=self.layout, add=add,
                                           dtype=None if add is not None else self.dtype)
